// linear.hip - rows times a weight held in 8-bit blocks, the rows quantised on the way.
//
//   out[i, :] = sum over k of blocks(x)[i, k] w[:, k]        (blocks(x), w: see blocks.hip)
//
// Three ways by the sizes: few rows read the weight once and split k over a workgroup's waves; many rows and few columns
// quantise each row's block in the registers of the wave that multiplies it, so x is read once and nothing is written but the
// result; everything else quantises x into the workspace and takes the tiled product.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "blocks.hpp"
#include "common.hpp"

namespace gsx_amd {

// Of a block's 128 k, a lane group g = lane / 16 holds 16 from 16 g on and 16 from 64 + 16 g on: one load of the four groups
// reads 64 bytes of each weight row in a piece.
__device__ inline int64_t piece_k(int64_t k0, int half, int lane) { return k0 + 64 * half + 16 * (lane / 16); }

// A lane's 32 elements of block k0 of a row. In a block that is cut, what lies past the last column is put right only when the
// block is used (cut_block): nothing waits for a load that is issued ahead.
template <typename T>
struct RawBlock {
    Raw<T, 8> v[4];
};

template <typename T>
__device__ inline void load_block(const T* __restrict__ row, int64_t k0, int64_t cols, int lane, RawBlock<T>& x) {
    if (cols >= 8) {
#pragma unroll
        for (int o = 0; o < 4; ++o)
            x.v[o] = load_raw<T, 8>(row + min(piece_k(k0, o / 2, lane) + 8 * (o & 1), cols - 8));
    } else {
#pragma unroll
        for (int o = 0; o < 4; ++o) x.v[o] = load_raw<T, 8>(row, piece_k(k0, o / 2, lane) + 8 * (o & 1), cols);
    }
}

template <typename T>
__device__ inline void cut_block(int64_t k0, int64_t cols, int lane, RawBlock<T>& x) {
    if (k0 + kBlock <= cols || cols < 8) return;
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        const int64_t over = piece_k(k0, o / 2, lane) + 8 * (o & 1) + 8 - cols;
        if (over > 0) x.v[o] = over < 8 ? shift_raw<T, 8>(x.v[o], (int)over) : Raw<T, 8>{};
    }
}

// The values that a row's block stands for, from the 32 that each of its four lanes holds; y[o] are those of v[o].
template <typename T>
__device__ inline void quantize_block(const RawBlock<T>& raw, v8bf (&y)[4]) {
    bool special;
    uint32_t top = largest_raw<T, 8, 4>(raw.v, special);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    const float scale = block_scale((uint32_t)(block_exponent(top) + 127));
#pragma unroll
    for (int o = 0; o < 4; ++o)
        y[o] = to_bf16((int)pack_raw<T, 8>(raw.v[o], 0, scale, special), (int)pack_raw<T, 8>(raw.v[o], 4, scale, special), scale);
}

// ---- few rows -------------------------------------------------------------------------------------------------------------
//
// A workgroup of up to 8 waves forms 16 J columns of out for up to 16 rows; wave w takes blocks w, w + waves, ... of k, so
// that together they read whole stretches of the weight's rows, and the waves' sums are joined through LDS. The rows of x
// are quantised into LDS first, `span` blocks of k at a time (all of them where they fit), while the weight's first block is
// on its way. Reading the weight bounds it: one row, 32768 x 4096, 135 MB in 28.6 us (4.7 TB/s).
constexpr int kFewRows = 16;
constexpr int kFewWaves = 8;
constexpr int kFewLeastWaves = 4;
constexpr int kFewBytes = 32768;  // of quantised rows in LDS

template <int J>
struct WeightBlock {
    v4i v[J][2];
    uint32_t exponent[J];
};

template <int J>
__device__ inline void load_weight(const BlockMatrix& w, const int64_t (&row)[J], int64_t kb, int64_t k, int lane,
                                   WeightBlock<J>& b) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint8_t* const p = w.values + row[j] * w.values_stride;
        if ((kb + 1) * kBlock <= k) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                b.v[j][half] = *reinterpret_cast<const v4i*>(p + piece_k(kb * kBlock, half, lane));
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) b.v[j][half] = load_values(p, piece_k(kb * kBlock, half, lane), k);
        }
        b.exponent[j] = w.exponents[row[j] * w.exponents_stride + kb];
    }
}

template <typename T, typename O, int J>
__global__ __launch_bounds__(64 * kFewWaves, 4) void linear_few_kernel(const T* __restrict__ x, int64_t x_stride, BlockMatrix w,
                                                                    int m, int64_t n, int64_t k, int span,
                                                                    O* __restrict__ out, int64_t out_stride) {
    extern __shared__ __attribute__((aligned(16))) uint8_t s_few[];
    v4f(*const s_acc)[J][64] = reinterpret_cast<v4f(*)[J][64]>(s_few);  // one for each wave
    uint8_t* const s_x = s_few + sizeof(v4f) * 64 * J * (blockDim.x / 64);  // [block][row][128], chunk c at place c ^ row % 8
    uint8_t* const s_e = s_x + (int64_t)span * m * kBlock;
    const int lane = threadIdx.x & 63, waves = blockDim.x / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t blocks = ceil_div(k, kBlock), tiles = ceil_div(n, 16 * J);
    const int x_row = min(lane & 15, m - 1);
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t n0 = t * 16 * J;
        int64_t row[J];
#pragma unroll
        for (int j = 0; j < J; ++j) row[j] = min(n0 + column_of<J>(j, lane & 15), n - 1);
        v4f acc[J];
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        WeightBlock<J> next;
        for (int64_t kb0 = 0; kb0 < blocks; kb0 += span) {
            const int64_t end = min(kb0 + span, blocks);
            if (kb0 + wave < end) load_weight<J>(w, row, kb0 + wave, k, lane, next);
            if (blocks > span || t == blockIdx.x) {
                __syncthreads();
                const int sub = threadIdx.x & 15;
                for (int i = threadIdx.x / 16; i < (int)(end - kb0) * m; i += blockDim.x / 16) {
                    const int64_t kb = kb0 + i / m;
                    const int r = i % m;
                    const int64_t col = kb * kBlock + sub * 8;
                    const Raw<T, 8> v[1] = {load_raw<T, 8>(x + r * x_stride, col, k)};
                    bool special;
                    uint32_t top = largest_raw<T, 8, 1>(v, special);
#pragma unroll
                    for (int off = 8; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 16));
                    const uint32_t e = (uint32_t)(block_exponent(top) + 127);
                    const float scale = block_scale(e);
                    *reinterpret_cast<uint2*>(s_x + i * kBlock + ((sub / 2) ^ (r & 7)) * 16 + (sub & 1) * 8) =
                        make_uint2(pack_raw<T, 8>(v[0], 0, scale, special), pack_raw<T, 8>(v[0], 4, scale, special));
                    if (sub == 0) s_e[i] = (uint8_t)e;
                }
                __syncthreads();
            }
            for (int64_t kb = kb0 + wave; kb < end; kb += waves) {
                const WeightBlock<J> now = next;
                if (kb + waves < end) load_weight<J>(w, row, kb + waves, k, lane, next);
                const int at = (int)(kb - kb0) * m + x_row;
                const float x_scale = block_scale(s_e[at]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const v4i q = *reinterpret_cast<const v4i*>(s_x + at * kBlock + ((4 * half + lane / 16) ^ (x_row & 7)) * 16);
                    const v8bf x0 = to_bf16(q[0], q[1], x_scale), x1 = to_bf16(q[2], q[3], x_scale);
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float scale = block_scale(now.exponent[j]);
                        const v4i u = now.v[j][half];
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(u[0], u[1], scale), x0, acc[j], 0, 0, 0);
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(u[2], u[3], scale), x1, acc[j], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) s_acc[wave][j][lane] = acc[j];
        __syncthreads();
        if (wave == 0) {
            for (int v = 1; v < waves; ++v)
#pragma unroll
                for (int j = 0; j < J; ++j) acc[j] += s_acc[v][j][lane];
            if ((lane & 15) < m) store_columns<J>(out + (lane & 15) * out_stride, n0 + (lane / 16) * (4 * J), n, acc);
        }
        __syncthreads();
    }
}

// ---- few columns ----------------------------------------------------------------------------------------------------------
//
// A wave takes 16 R rows and all (up to 16 TN) columns; x is read once, straight into registers, a block ahead. The weight lies
// in LDS for the workgroup's four waves, all of it where it fits (kHeadBytes) and is then read once for all the tiles of a
// workgroup, else a block of 128 k at a time; each wave converts it. The result passes through LDS, 16 rows of a wave at a
// time, and leaves in whole stretches of its rows. 307200 x 128 to 150 columns: 46 us for 171 MB, 3.7 TB/s; quantising and
// converting in two or three waves a SIMD is about as long as the memory's time and only partly hides in it.
constexpr int kHeadThreads = 256;
constexpr int kHeadBytes = 49152;
template <int TN>
constexpr int kHeadRows = TN > 4 ? 16 : 32;  // of a wave: more hide less of the loads' time for want of registers
template <typename O, int TN>
constexpr int kHeadPitch = 16 * TN * (int)sizeof(O) + 16;
template <int TN>
constexpr int kHeadResident = kHeadBytes / (16 * TN * kBlock);  // blocks of k that fit

template <typename T, typename O, int TN>
__global__ __launch_bounds__(kHeadThreads, 2) void linear_head_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                      BlockMatrix w, int64_t m, int64_t n, int64_t k,
                                                                      int slots, O* __restrict__ out, int64_t out_stride) {
    constexpr int R = kHeadRows<TN> / 16, kRows = 16 * TN, kWaves = kHeadThreads / 64;
    constexpr int kOct = 8;  // columns a lane stores at once
    extern __shared__ __attribute__((aligned(16))) uint8_t s_head[];  // slots for blocks of the weight, their exponents
    uint8_t* const s_w = s_head;
    uint8_t* const s_e = s_head + slots * kRows * kBlock;
    __shared__ __attribute__((aligned(16))) uint8_t s_out[kWaves][16 * kHeadPitch<O, TN>];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int64_t blocks = ceil_div(k, kBlock), tiles = ceil_div(m, kHeadRows<TN> * kWaves);
    const bool resident = blocks <= slots;
    const auto stage = [&](int64_t kb, int slot) {
        for (int i = threadIdx.x; i < kRows * 8; i += kHeadThreads) {
            const int row = i / 8, chunk = i % 8;
            const int64_t source = min((int64_t)row, n - 1);
            *reinterpret_cast<v4i*>(s_w + (slot * kRows + row) * kBlock + ((chunk ^ swizzle_b<TN>(row)) * 16)) =
                load_values(w.values + source * w.values_stride, kb * kBlock + chunk * 16, k);
            if (chunk == 0) s_e[slot * kRows + row] = w.exponents[source * w.exponents_stride + kb];
        }
    };
    RawBlock<T> next[R];
    const auto load = [&](int64_t tile, int64_t kb) {
        const int64_t m0 = (tile * kWaves + wave) * kHeadRows<TN>;
#pragma unroll
        for (int r = 0; r < R; ++r)
            load_block<T>(x + min(m0 + r * 16 + (lane & 15), m - 1) * x_stride, kb * kBlock, k, lane, next[r]);
    };
    if ((int64_t)blockIdx.x < tiles && blocks > 0) load(blockIdx.x, 0);
    if (resident) {
        for (int64_t kb = 0; kb < blocks; ++kb) stage(kb, (int)kb);
        __syncthreads();
    }
    // lanes of a stretch of 8 columns, a power of two, and the rows that 64 lanes cover
    int across = 1;
    while (across * kOct < n) across *= 2;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t m0 = (t * kWaves + wave) * kHeadRows<TN>;
        v4f acc[R][TN];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[r][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t kb = 0; kb < blocks; ++kb) {
            int slot = (int)kb;
            if (!resident) {
                slot = 0;
                __syncthreads();
                stage(kb, 0);
                __syncthreads();
            }
            v8bf vx[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                cut_block<T>(kb * kBlock, k, lane, next[r]);
                quantize_block<T>(next[r], vx[r]);
            }
            if (kb + 1 < blocks) load(t, kb + 1);
            else if (t + gridDim.x < tiles) load(t + gridDim.x, 0);
            const uint8_t* const values = s_w + slot * kRows * kBlock;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int row = column_of<TN>(j, lane & 15);
                const float scale = block_scale(s_e[slot * kRows + row]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const v4i q = *reinterpret_cast<const v4i*>(
                        values + row * kBlock + (((4 * half + lane / 16) ^ swizzle_b<TN>(row)) * 16));
                    const v8bf w0 = to_bf16(q[0], q[1], scale), w1 = to_bf16(q[2], q[3], scale);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, vx[r][2 * half], acc[r][j], 0, 0, 0);
                        acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, vx[r][2 * half + 1], acc[r][j], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            uint8_t* const mine = s_out[wave];
            wave_lds_sync();
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                Vec<O, 4> q;
#pragma unroll
                for (int i = 0; i < 4; ++i) q.v[i] = from_float<O>(acc[r][j][i]);
                *reinterpret_cast<Vec<O, 4>*>(mine + (lane & 15) * kHeadPitch<O, TN> +
                                              ((lane / 16) * 4 * TN + 4 * j) * sizeof(O)) = q;
            }
            wave_lds_sync();
            const int col = lane % across * kOct;
            for (int i = lane / across; i < 16; i += 64 / across) {
                const int64_t row = m0 + r * 16 + i;
                if (row < m && col + kOct <= n)
                    *reinterpret_cast<Octet<O>*>(out + row * out_stride + col) =
                        *reinterpret_cast<const Octet<O>*>(mine + i * kHeadPitch<O, TN> + col * sizeof(O));
            }
            if (n % kOct != 0) {  // the last columns of eight rows at a time, one a lane
                const int64_t last = n / kOct * kOct + lane % kOct;
                for (int i = lane / kOct; i < 16; i += 64 / kOct) {
                    const int64_t row = m0 + r * 16 + i;
                    if (row < m && last < n)
                        out[row * out_stride + last] = reinterpret_cast<const O*>(mine + i * kHeadPitch<O, TN>)[last];
                }
            }
        }
    }
}

// ---- gradient of the weight, narrow layers ----------------------------------------------------------------------------------
//
//   gw[i, j] = sum over rows r of blocks(dy^T)[i, r] blocks(x^T)[j, r]
//
// A workgroup takes a stretch of blocks of 128 rows. Of each it reads dy and x once, finds the columns' maxima, quantises the
// columns into LDS (a column's 128 values in a row of kWeightPitch bytes, so that a read of 16 columns meets 16 different banks)
// and multiplies them, 2 x 4 waves with NT x KT tiles of 16 x 16 each; the next block's rows are on their way meanwhile. The
// stretches' sums are joined by another launch. Quantised copies of dy^T and x^T, written and read again, would double what is
// moved. 307200 x 150 x 128 of bf16: 69 us for 171 MB, 2.5 TB/s. Registers leave one workgroup a CU, whose phases (maxima,
// quantising, products) stand between barriers (the waves wait for 44% of their time, the vector units are busy for 33%, the
// matrix units for 8%): with a second block's rows on their way it is no faster; with 16 waves 4% for 16-bit types, whose float32
// form spills.
constexpr int kWeightThreads = 512;
constexpr int kWeightPitch = 144;
constexpr int kWeightPatches = 3;  // of 8 rows by 4 columns a thread holds: up to 96 quads of columns
constexpr int64_t kWeightMostColumns = 4 * 96 - 6;

template <typename T, int NT, int KT>
__global__ __launch_bounds__(kWeightThreads) void linear_weight_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                       const T* __restrict__ dy, int64_t dy_stride,
                                                                       int64_t m, int n, int k,
                                                                       float* __restrict__ partial) {
    constexpr int kN = 32 * NT, kK = 64 * KT;
    __shared__ __attribute__((aligned(16))) uint8_t s_q[(kN + kK) * kWeightPitch];
    __shared__ uint32_t s_top[kN + kK];
    __shared__ uint8_t s_e[kN + kK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, wn = wave / 4, wk = wave % 4;
    const int64_t blocks = ceil_div(m, kBlock);
    const int64_t first = blocks * blockIdx.x / gridDim.x, last = blocks * (blockIdx.x + 1) / gridDim.x;
    // patch u of a thread: 8 rows from r0 on of the quad of columns at `column` of LDS (dy's columns before x's). A last quad that
    // is cut is read from `back` columns further left, so that no read leaves its row.
    const int dy_quads = (n + 3) / 4, quads = dy_quads + (k + 3) / 4;
    int r0[kWeightPatches], column[kWeightPatches], back[kWeightPatches];
    bool some[kWeightPatches];
    const T* from[kWeightPatches];
    int64_t stride[kWeightPatches];
#pragma unroll
    for (int u = 0; u < kWeightPatches; ++u) {
        const int p = threadIdx.x + u * kWeightThreads, q = p % quads;
        const bool is_dy = q < dy_quads;
        const int c = (is_dy ? q : q - dy_quads) * 4;
        r0[u] = p / quads * 8;
        column[u] = is_dy ? c : kN + c;
        some[u] = r0[u] < kBlock;
        back[u] = max(0, c + 4 - (is_dy ? n : k));
        from[u] = (is_dy ? dy : x) + (c - back[u]);
        stride[u] = is_dy ? dy_stride : x_stride;
    }
    Raw<T, 4> raw[kWeightPatches][8];
    const auto load = [&](int64_t block) {
#pragma unroll
        for (int u = 0; u < kWeightPatches; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t row = block * kBlock + r0[u] + i;
                raw[u][i] = {};
                if (some[u] && row < m) raw[u][i] = load_raw<T, 4>(from[u] + row * stride[u]);
            }
    };
    v4f acc[NT][KT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < KT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (first < last) load(first);
    for (int64_t block = first; block < last; ++block) {
        // what follows from these is worked out anew for each block: kept, it takes the registers of the rows
#pragma unroll
        for (int u = 0; u < kWeightPatches; ++u) asm volatile("" : "+v"(column[u]), "+v"(r0[u]));
        for (int i = threadIdx.x; i < kN + kK; i += kWeightThreads) s_top[i] = 0;
        __syncthreads();  // and the block before has been multiplied
        bool special[kWeightPatches];
#pragma unroll
        for (int u = 0; u < kWeightPatches; ++u) {
            if (!some[u]) continue;
            if (back[u] != 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[u][i] = shift_raw<T, 4>(raw[u][i], back[u]);
            }
            uint32_t top[4];
            special[u] = patch_tops<T>(raw[u], top);
#pragma unroll
            for (int c = 0; c < 4; ++c) atomicMax(&s_top[column[u] + c], top[c]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kWeightPatches; ++u) {
            if (!some[u]) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t e = (uint32_t)(block_exponent(s_top[column[u] + c]) + 127);
                *reinterpret_cast<uint2*>(s_q + (column[u] + c) * kWeightPitch + r0[u]) =
                    patch_column<T>(raw[u], c, block_scale(e), special[u]);
                if (r0[u] == 0) s_e[column[u] + c] = (uint8_t)e;
            }
        }
        __syncthreads();
        if (block + 1 < last) load(block + 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int at = (lane / 16) * 16 + 64 * half;
            v8bf vx[KT][2];
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const int c = kN + (wk * KT + j) * 16 + (lane & 15);
                const v4i q = *reinterpret_cast<const v4i*>(s_q + c * kWeightPitch + at);
                const float scale = block_scale(s_e[c]);
                vx[j][0] = to_bf16(q[0], q[1], scale);
                vx[j][1] = to_bf16(q[2], q[3], scale);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int c = (wn * NT + i) * 16 + (lane & 15);
                const v4i q = *reinterpret_cast<const v4i*>(s_q + c * kWeightPitch + at);
                const float scale = block_scale(s_e[c]);
                const v8bf y0 = to_bf16(q[0], q[1], scale), y1 = to_bf16(q[2], q[3], scale);
#pragma unroll
                for (int j = 0; j < KT; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vx[j][0], y0, acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vx[j][1], y1, acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    // the result's rows are columns of dy (lane % 16), its columns four of x a lane
    float* const to = partial + (int64_t)blockIdx.x * n * k;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int row = (wn * NT + i) * 16 + (lane & 15);
        if (row >= n) continue;
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            const v4f one[1] = {acc[i][j]};
            store_columns<1>(to + (int64_t)row * k, (wk * KT + j) * 16 + (lane / 16) * 4, k, one);
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

constexpr int64_t kHeadMostColumns = 256;
constexpr int kHeadMostBlocks = 6;

enum class LinearWay { kFew, kHead, kTiles };

// Few rows while the quantised rows fit a workgroup's LDS (k = n = 8192: 1 row 18 us against 24 through the tiled product, 4 rows
// 21 against 24.5, 8 rows, which do not fit, 28 against 24.5) and no wave's sum is longer than kSumMostBlocks (one row, k =
// 300000: 64 columns 204 us and 1024 257 in longer sums, 19 and 96 through the tiled product). Few columns up to some blocks of
// k: three (65536 x 150 x 384: 37 us either way, 512 47 against 44); up to 64 columns leave room for the weight's six in LDS,
// which pays with many rows (40 columns, k = 768: 307200 rows 135 us against 186, 8000 rows 27 against 20); more than 192 columns
// one, two with few rows (250 columns, k = 256: 307200 rows 154 us against 127, 2000 rows 17 against 19).
LinearWay linear_way(int64_t m, int64_t n, int64_t k) {
    const int64_t blocks = ceil_div(k, kBlock);
    if (m <= kFewRows && (m <= 2 || m * blocks * kBlock <= kFewBytes) && blocks <= kFewLeastWaves * kSumMostBlocks)
        return LinearWay::kFew;
    const bool many = m >= 32768;
    const int most = n <= 64 ? (many ? kHeadMostBlocks : 3) : n <= 192 ? 3 : many ? 1 : 2;
    return n <= kHeadMostColumns && k <= most * kBlock ? LinearWay::kHead : LinearWay::kTiles;
}

// The quantised rows in the workspace, rounded up for what follows them.
int64_t linear_rows_bytes(int64_t m, int64_t k) {
    const int64_t blocks = ceil_div(k, kBlock);
    return ceil_div(m * (blocks * kBlock + ceil_div(blocks, 4) * 4), 256) * 256;
}

template <typename T, typename O, int TN>
gsx_hip_status launch_head(const T* x, int64_t x_stride, const BlockMatrix& w, int64_t m, int64_t n, int64_t k, O* out,
                           int64_t out_stride, hipStream_t stream) {
    // as many workgroups as run at once, so that all take the same share (307200 x 128 to 150 columns: 768 of them 48 us, 512 or
    // 1024 53); registers and LDS decide how many a CU takes, which is asked once for each kernel and number of slots
    const int64_t tiles = ceil_div(m, kHeadRows<TN> * (kHeadThreads / 64)), blocks = ceil_div(k, kBlock);
    const int slots = blocks <= kHeadResident<TN> ? (int)(blocks > 0 ? blocks : 1) : 1;
    const int lds = slots * 16 * TN * (kBlock + 1);
    static std::atomic<int> a_cu[kHeadMostBlocks + 1];
    int each = a_cu[slots].load(std::memory_order_relaxed);
    if (each == 0) {
        const hipError_t e =
            hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, linear_head_kernel<T, O, TN>, kHeadThreads, lds);
        if (e != hipSuccess || each < 1) {
            (void)hipGetLastError();  // it is returned here
            return fields_fail(e != hipSuccess ? (gsx_hip_status)e : GSX_HIP_ERROR_INVALID_STATE, "linear: workgroups of a CU");
        }
        a_cu[slots].store(each, std::memory_order_relaxed);
    }
    const int64_t most = (int64_t)each * 256;
    hipLaunchKernelGGL((linear_head_kernel<T, O, TN>), dim3((unsigned)(tiles < most ? tiles : most)), dim3(kHeadThreads),
                       (unsigned)lds, stream, x, x_stride, w, m, n, k, slots, out, out_stride);
    return fields_launched("linear launch");
}

// Stretches of rows that the weight's gradient of a narrow layer is split into; 0: the layer is not narrow, or too short for its
// partial sums to be few beside what is read.
int64_t weight_stretches(int32_t x_type, int32_t grad_type, int64_t m, int64_t n, int64_t k) {
    if (x_type != grad_type) return 0;  // the kernel is built for rows of one type
    if (n < 4 || k < 4 || n + k > kWeightMostColumns || n > (k <= 128 ? 256 : 128) || k > 256 || m < 8192) return 0;
    const int64_t blocks = ceil_div(m, kBlock);
    return blocks < 256 ? blocks : std::max<int64_t>(256, ceil_div(blocks, kSumMostBlocks));
}

struct WeightBlocks {  // workspace of the general way: byte offsets
    int64_t blocks, words, dy_values, dy_exponents, x_values, x_exponents, rest;
    WeightBlocks(int64_t m, int64_t n, int64_t k) {
        blocks = ceil_div(m, kBlock);
        words = ceil_div(blocks, 4) * 4;
        int64_t at = 0;
        const auto take = [&](int64_t size) {
            const int64_t here = at;
            at += ceil_div(size, 256) * 256;
            return here;
        };
        dy_values = take(n * blocks * kBlock);
        dy_exponents = take(n * words);
        x_values = take(k * blocks * kBlock);
        x_exponents = take(k * words);
        rest = at;
    }
};

}  // namespace

extern "C" {

size_t gsx_hip_linear_temp_bytes(int64_t m, int64_t n, int64_t k) {
    if (!product_sizes(m, n, k) || linear_way(m, n, k) != LinearWay::kTiles) return 0;
    return (size_t)linear_rows_bytes(m, k) + gsx_hip_blocks_matmul_temp_bytes(m, n, k);
}

gsx_hip_status gsx_hip_linear_forward(const void* x, int32_t x_type, int64_t x_stride, const uint8_t* w_values,
                                      int64_t w_values_stride, const uint8_t* w_exponents, int64_t w_exponents_stride,
                                      int64_t m, int64_t n, int64_t k, void* out, int32_t out_type, int64_t out_stride,
                                      void* temp, hipStream_t stream) {
    if (!known_type(x_type) || !known_type(out_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "linear: rows are f32, bf16 or f16");
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "linear: at most 2^31 - 1 rows and columns and 2^27 summands");
    if (!rows_fit(m, x_stride, k) || !rows_fit(m, out_stride, n))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "linear: strides must be at least the rows' lengths");
    const gsx_hip_status wrong = block_matrix_check(w_values, w_exponents, n, k, w_values_stride, w_exponents_stride);
    if (wrong != GSX_HIP_SUCCESS) return wrong;
    if (m == 0 || n == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || (k > 0 && x == nullptr) || !aligned_to(out, type_bytes(out_type)) ||
        !aligned_to(x, type_bytes(x_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "linear: rows must be non-null and aligned to their elements");
    const LinearWay way = linear_way(m, n, k);
    if (way == LinearWay::kTiles) {
        if (k > 0 && (temp == nullptr || !aligned_to(temp, 16)))
            return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "linear: the workspace must be non-null and 16-byte aligned");
        if (w_values_stride >= kMostStride)
            return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "linear: a wide layer's value rows lie less than 2^28 bytes apart");
        const int64_t blocks = ceil_div(k, kBlock), words = ceil_div(blocks, 4) * 4;
        uint8_t* const values = static_cast<uint8_t*>(temp);
        uint8_t* const exponents = values + m * blocks * kBlock;
        const gsx_hip_status st = gsx_hip_blocks_quantize(x, x_type, m, k, x_stride, 0, values, blocks * kBlock, exponents,
                                                          words, stream);
        if (st != GSX_HIP_SUCCESS) return st;
        return gsx_hip_blocks_matmul(values, blocks * kBlock, exponents, words, w_values, w_values_stride, w_exponents,
                                     w_exponents_stride, m, n, k, out, out_type, out_stride,
                                     values + linear_rows_bytes(m, k), stream);
    }
    const BlockMatrix w = {w_values, w_exponents, w_values_stride, w_exponents_stride};
    return with_type(x_type, [&](auto tx) {
        return with_type(out_type, [&](auto to) {
            using T = decltype(tx);
            using O = decltype(to);
            const T* const from = static_cast<const T*>(x);
            O* const result = static_cast<O*>(out);
            if (way == LinearWay::kFew) {
                // waves enough for the GPU: 32 columns a workgroup where that leaves 1024 of them, else 16, and up to 8
                // waves over k
                const int64_t blocks = ceil_div(k, kBlock), strips = ceil_div(n, 16);
                const int j = strips >= 2048 ? 2 : 1;
                int64_t waves = kFewLeastWaves;
                while (waves < kFewWaves && waves < blocks && ceil_div(strips, j) * waves < 4096) waves *= 2;
                const int64_t groups = ceil_div(strips, j);
                int64_t span = kFewBytes / kBlock / m;
                if (span > blocks) span = blocks;
                const int64_t lds = waves * j * 1024 + span * m * (kBlock + 1);
                hipLaunchKernelGGL((j == 2 ? linear_few_kernel<T, O, 2> : linear_few_kernel<T, O, 1>),
                                   dim3((unsigned)(groups < 1024 ? groups : 1024)), dim3((unsigned)waves * 64),
                                   (unsigned)lds, stream, from, x_stride, w, (int)m, n, k, (int)span, result, out_stride);
                return fields_launched("linear launch");
            }
            if (n <= 64) return launch_head<T, O, 4>(from, x_stride, w, m, n, k, result, out_stride, stream);
            if (n <= 128) return launch_head<T, O, 8>(from, x_stride, w, m, n, k, result, out_stride, stream);
            if (n <= 192) return launch_head<T, O, 12>(from, x_stride, w, m, n, k, result, out_stride, stream);
            return launch_head<T, O, 16>(from, x_stride, w, m, n, k, result, out_stride, stream);
        });
    });
}

size_t gsx_hip_linear_backward_weight_temp_bytes(int32_t x_type, int32_t grad_type, int64_t m, int64_t n, int64_t k) {
    if (!product_sizes(m, n, k) || m > kMostSummands || n == 0 || k == 0) return 0;
    const int64_t stretches = weight_stretches(x_type, grad_type, m, n, k);
    if (stretches > 0) return (size_t)(stretches * n * k * 4);
    return (size_t)WeightBlocks(m, n, k).rest + gsx_hip_blocks_matmul_temp_bytes(n, k, m);
}

gsx_hip_status gsx_hip_linear_backward_weight(const void* x, int32_t x_type, int64_t x_stride, const void* grad_out,
                                              int32_t grad_type, int64_t grad_stride, int64_t m, int64_t n, int64_t k,
                                              float* grad_weight, int64_t weight_stride, void* temp, hipStream_t stream) {
    if (!known_type(x_type) || !known_type(grad_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "linear backward: rows are f32, bf16 or f16");
    if (!product_sizes(m, n, k) || m > kMostSummands)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "linear backward: at most 2^27 rows, 2^31 - 1 and 2^27 columns");
    if (!rows_fit(m, x_stride, k) || !rows_fit(m, grad_stride, n) || !rows_fit(n, weight_stride, k))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "linear backward: strides must be at least the rows' lengths");
    if (n == 0 || k == 0) return GSX_HIP_SUCCESS;
    if (grad_weight == nullptr || !aligned_to(grad_weight, 4) ||
        (m > 0 && (x == nullptr || grad_out == nullptr || temp == nullptr)) || !aligned_to(x, type_bytes(x_type)) ||
        !aligned_to(grad_out, type_bytes(grad_type)) || !aligned_to(temp, 16))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "linear backward: rows and workspace must be non-null and aligned to their elements");
    const int64_t stretches = weight_stretches(x_type, grad_type, m, n, k);
    if (stretches == 0) {
        const WeightBlocks at(m, n, k);
        uint8_t* const base = static_cast<uint8_t*>(temp);
        gsx_hip_status st = gsx_hip_blocks_quantize(grad_out, grad_type, m, n, grad_stride, 1, base + at.dy_values,
                                                    at.blocks * kBlock, base + at.dy_exponents, at.words, stream);
        if (st != GSX_HIP_SUCCESS) return st;
        st = gsx_hip_blocks_quantize(x, x_type, m, k, x_stride, 1, base + at.x_values, at.blocks * kBlock,
                                     base + at.x_exponents, at.words, stream);
        if (st != GSX_HIP_SUCCESS) return st;
        return gsx_hip_blocks_matmul(base + at.dy_values, at.blocks * kBlock, base + at.dy_exponents, at.words,
                                     base + at.x_values, at.blocks * kBlock, base + at.x_exponents, at.words, n, k, m,
                                     grad_weight, GSX_HIP_DTYPE_F32, weight_stride, base + at.rest, stream);
    }
    return with_type(x_type, [&](auto t) {
        using T = decltype(t);
        float* const partial = static_cast<float*>(temp);
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)stretches), dim3(kWeightThreads), 0, stream, static_cast<const T*>(x),
                               x_stride, static_cast<const T*>(grad_out), grad_stride, m, (int)n, (int)k, partial);
        };
        if (k <= 128) {
            if (n <= 128) go(linear_weight_kernel<T, 4, 2>);
            else if (n <= 192) go(linear_weight_kernel<T, 6, 2>);
            else go(linear_weight_kernel<T, 8, 2>);
        } else {
            go(linear_weight_kernel<T, 4, 4>);
        }
        const gsx_hip_status st = fields_launched("linear backward launch");
        return st != GSX_HIP_SUCCESS ? st : join_products(partial, n, k, stretches, grad_weight, weight_stride, stream);
    });
}

}  // extern "C"

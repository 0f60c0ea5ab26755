// linear4.hip - rows times a weight held in 4-bit blocks, the rows quantised on the way.
//
//   out[i, :] = sum over k of blocks(x)[i, k] w[:, k]        (blocks(x), w: see blocks4.hip)
//
// Three ways by the sizes: few rows read the weight once and split k over a workgroup's waves; many rows and few columns
// quantise each row's blocks in the registers of the lane that multiplies them, so x is read once and nothing is written but the
// result; everything else quantises x into the workspace and takes the tiled product.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "blocks4.hpp"
#include "common.hpp"

namespace gsx_amd {

// A lane's block of 32 elements of a row, zeros past the last column, as it lies in memory.
template <typename T>
struct RawBlock4 {
    Raw<T, 8> v[4];
};

template <typename T>
__device__ inline void load_block4_of(const T* __restrict__ row, int64_t kb, int64_t cols, RawBlock4<T>& x) {
    if ((kb + 1) * kBlock4 <= cols) {
#pragma unroll
        for (int o = 0; o < 4; ++o) x.v[o] = load_raw<T, 8>(row + kb * kBlock4 + 8 * o);
        return;
    }
#pragma unroll
    for (int o = 0; o < 4; ++o) x.v[o] = load_raw<T, 8>(row, kb * kBlock4 + 8 * o, cols);
}

// The same block quantised: values and exponent byte.
template <typename T>
__device__ inline v4i quantize_block4(const RawBlock4<T>& x, uint32_t& exponent) {
    bool special;
    const uint32_t top = largest_raw<T, 8, 4>(x.v, special);
    exponent = special ? kNoScale : (uint32_t)(block4_exponent(top) + 127);
    const float scale = block_scale(special ? 127u : exponent);
    v4i q;
#pragma unroll
    for (int o = 0; o < 4; ++o) q[o] = (int)pack4_raw<T, 8>(x.v[o], 0, scale);
    return q;
}

// Four blocks of a row, one for each lane group, as loads of 64 bytes in a piece bring them: load p of group g brings piece 4 p + g
// of 16 bytes. (Each lane's block in 64 or 128 bytes of its own meets every line four or eight times; 307200 rows of 128 bf16, 150
// columns: 41.9 us, so 39.6.) The groups then exchange pieces, a transposition of four by four.
template <typename T>
__device__ inline void load_quad4_of(const T* __restrict__ row, int64_t quad, int group, RawBlock4<T>& x) {
    constexpr int kPieces = 2 * (int)sizeof(T), kEach = 16 / (int)sizeof(T);
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        const Raw<T, kEach> y = load_raw<T, kEach>(row + quad * 4 * kBlock4 + (4 * p + group) * kEach);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[p * 4 / Raw<T, 8>::kWords].w[p * 4 % Raw<T, 8>::kWords + i] = y.w[i];
    }
}

template <typename T>
__device__ inline void exchange_quad4(RawBlock4<T>& x) {
    constexpr int kPieces = 2 * (int)sizeof(T), kTogether = kPieces / 4, kWords = Raw<T, 8>::kWords;
    uint32_t in[4][4 * kTogether];  // pieces kTogether P .. of load order
#pragma unroll
    for (int i = 0; i < 4 * kPieces; ++i) in[i / (4 * kTogether)][i % (4 * kTogether)] = x.v[i / kWords].w[i % kWords];
#pragma unroll
    for (int i = 0; i < 4 * kTogether; ++i) {
        const auto a = __builtin_amdgcn_permlane16_swap(in[0][i], in[1][i], false, false);
        const auto b = __builtin_amdgcn_permlane16_swap(in[2][i], in[3][i], false, false);
        const auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
        const auto d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
        in[0][i] = c[0];
        in[2][i] = c[1];
        in[1][i] = d[0];
        in[3][i] = d[1];
    }
    // piece 4 e + h of the lane's block came from group h
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[q * 4 / kWords].w[q * 4 % kWords + i] = in[q % 4][q / 4 * 4 + i];
}

// ---- few rows -------------------------------------------------------------------------------------------------------------
//
// A workgroup of up to 8 waves forms 16 columns of out for up to 16 rows; wave w takes chunks w, w + waves, ... of 512 k, of
// which a lane of group g = lane / 16 holds blocks 4 g to 4 g + 3 (64 bytes in a piece, their exponents one word), one for each of
// four instructions. The waves' sums are joined through LDS. The rows of x are quantised into LDS first, `span` chunks at a time,
// while the weight's first chunk is on its way.
constexpr int kFewRows4 = 16;
constexpr int kFewWaves4 = 8;
constexpr int kChunk4 = 16;          // blocks of a chunk
constexpr int kFewBytes4 = 49152;    // of quantised rows in LDS
constexpr int kFewPad4 = 16;         // bytes between rows there, so that rows meet different banks

struct FewShape {
    int span;  // chunks
    __host__ __device__ int values_pitch() const { return span * kChunk4 * 16 + kFewPad4; }
    __host__ __device__ int exponents_pitch() const { return span * kChunk4 + 4; }
};

struct WeightChunk4 {
    v4i v[4];
    uint32_t exponents;
};

__device__ inline WeightChunk4 load_chunk4(const uint8_t* values, const uint8_t* exponents, int chunk, int blocks, int group) {
    const int kb = chunk * kChunk4 + group * 4;
    WeightChunk4 c;
    if ((chunk + 1) * kChunk4 <= blocks) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c.v[s] = *reinterpret_cast<const v4i*>(values + (kb + s) * 16);
        c.exponents = reinterpret_cast<const uint32_t*>(exponents)[chunk * 4 + group];
    } else {  // x is 0 past the last k, whatever is read again here
#pragma unroll
        for (int s = 0; s < 4; ++s) c.v[s] = *reinterpret_cast<const v4i*>(values + min(kb + s, blocks - 1) * 16);
        c.exponents = load_exponents4(exponents, chunk * 4 + group, blocks);
    }
    return c;
}

template <typename T, typename O>
__global__ __launch_bounds__(64 * kFewWaves4, 4) void linear4_few_kernel(const T* __restrict__ x, int64_t x_stride, BlockMatrix w,
                                                                         int m, int64_t n, int64_t k, FewShape shape,
                                                                         O* __restrict__ out, int64_t out_stride) {
    extern __shared__ __attribute__((aligned(16))) uint8_t s_few4[];
    v4f(*const s_acc)[64] = reinterpret_cast<v4f(*)[64]>(s_few4);  // one for each wave
    uint8_t* const s_x = s_few4 + sizeof(v4f) * 64 * (blockDim.x / 64);
    uint8_t* const s_e = s_x + m * shape.values_pitch();
    const int lane = threadIdx.x & 63, group = lane / 16, waves = blockDim.x / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int blocks = (int)ceil_div(k, kBlock4), chunks = (blocks + kChunk4 - 1) / kChunk4;
    const int64_t tiles = ceil_div(n, 16);
    const int x_row = min(lane & 15, m - 1);
    const bool held = chunks <= shape.span;  // all of x in LDS
    const uint8_t *values, *exponents;       // the lane's row of the weight
    const auto turn_to = [&](int64_t tile) {
        const int64_t row = min(tile * 16 + (lane & 15), n - 1);
        values = w.values + row * w.values_stride;
        exponents = w.exponents + row * w.exponents_stride;
    };
    WeightChunk4 next;
    turn_to(blockIdx.x);
    if ((int64_t)blockIdx.x < tiles && wave < chunks) next = load_chunk4(values, exponents, wave, blocks, group);
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c0 = 0; c0 < chunks; c0 += shape.span) {
            const int end = min(c0 + shape.span, chunks);
            if (c0 > 0 && c0 + wave < end) next = load_chunk4(values, exponents, c0 + wave, blocks, group);
            if (!held || t == blockIdx.x) {
                __syncthreads();
                const int here = (end - c0) * kChunk4;  // whole chunks: zeros behind the last block
                for (int i = threadIdx.x; i < here * m; i += blockDim.x) {
                    const int r = i / here, b = i % here;
                    RawBlock4<T> raw;
                    load_block4_of<T>(x + r * x_stride, c0 * kChunk4 + b, k, raw);
                    uint32_t e;
                    *reinterpret_cast<v4i*>(s_x + r * shape.values_pitch() + b * 16) = quantize_block4<T>(raw, e);
                    s_e[r * shape.exponents_pitch() + b] = (uint8_t)e;
                }
                __syncthreads();
            }
            for (int c = c0 + wave; c < end; c += waves) {
                const WeightChunk4 now = next;
                if (c + waves < end) next = load_chunk4(values, exponents, c + waves, blocks, group);
                const int at = (c - c0) * kChunk4 + group * 4;
                const uint32_t e = *reinterpret_cast<const uint32_t*>(s_e + x_row * shape.exponents_pitch() + at);
                v4i q[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) q[s] = *reinterpret_cast<const v4i*>(s_x + x_row * shape.values_pitch() + (at + s) * 16);
                acc = multiply4<0, 0>(now.v[0], q[0], acc, now.exponents, e);
                acc = multiply4<1, 1>(now.v[1], q[1], acc, now.exponents, e);
                acc = multiply4<2, 2>(now.v[2], q[2], acc, now.exponents, e);
                acc = multiply4<3, 3>(now.v[3], q[3], acc, now.exponents, e);
            }
        }
        if (t + gridDim.x < tiles) {  // on its way while the waves are joined
            turn_to(t + gridDim.x);
            if (wave < chunks) next = load_chunk4(values, exponents, wave, blocks, group);
        }
        s_acc[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
            for (int v = 1; v < waves; ++v) acc += s_acc[v][lane];
            const v4f one[1] = {acc};
            if ((lane & 15) < m) store_columns<1>(out + (lane & 15) * out_stride, t * 16 + group * 4, n, one);
        }
        __syncthreads();
    }
}

// ---- few columns ----------------------------------------------------------------------------------------------------------
//
// A wave takes 16 R rows and all (up to 16 TN) columns, 128 k at a time: lane l holds block l / 16 of row l % 16, loads it, finds
// its largest value and quantises it without another lane's help. The weight lies in LDS for the workgroup's four waves and is read
// once for all the tiles of a workgroup; block b of its row r lies at place b ^ r % 4 of a group of four, so that the sixteen rows
// of a read meet different banks. The result passes through LDS, 16 rows of a wave at a time: where rows of out follow one another
// without a gap, as one stretch. The stores pass the caches by: 307200 x 150 x 128 in float32 76 us with them, 63 without.
constexpr int kHeadThreads4 = 256;
constexpr int kHeadWaves4 = kHeadThreads4 / 64;
template <typename T, int TN>
constexpr int kHeadRows4 = sizeof(T) == 4 || TN > 10 ? 16 : 32;  // of a wave: what the registers hold
constexpr int kHeadBytes4 = 65536;   // of the weight in LDS

// Elements of a row of the result in LDS: n, for one stretch, unless rows would meet in the same banks.
template <typename O>
__host__ __device__ inline int head4_pitch(int64_t n, int64_t out_stride) {
    return out_stride == n && n * (int64_t)sizeof(O) % 128 != 0 ? (int)n : (int)((n + 7) / 8 * 8 + 8);
}

template <typename T, typename O, int TN>
__global__ __launch_bounds__(kHeadThreads4, 2) void linear4_head_kernel(const T* __restrict__ x, int64_t x_stride, BlockMatrix w,
                                                                        int64_t m, int n, int64_t k, O* __restrict__ out,
                                                                        int64_t out_stride) {
    constexpr int kRows = kHeadRows4<T, TN>, R = kRows / 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_head4[];
    const int lane = threadIdx.x & 63, group = lane / 16, wave = threadIdx.x / 64;
    const int blocks = (int)ceil_div(k, kBlock4), quads = (int)ceil_div(blocks, 4), columns = ((n + 15) / 16) * 16;
    const int64_t tiles = ceil_div(m, kRows * kHeadWaves4);
    uint8_t* const s_w = s_head4;                             // [quad][column][4 blocks]
    uint8_t* const s_e = s_w + quads * columns * 64;          // [quad][column] words
    const int pitch = head4_pitch<O>(n, out_stride);
    O* const s_out = reinterpret_cast<O*>(s_e + quads * columns * 4) + wave * 16 * pitch;
    constexpr int kOct = 16 / (int)sizeof(O);
    const int across = (n + kOct - 1) / kOct, first_row = lane / across, first_piece = lane % across;  // vectors of a row
    RawBlock4<T> next[R];
    const auto load = [&](int64_t tile, int quad) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = min((tile * kHeadWaves4 + wave) * kRows + r * 16 + (lane & 15), m - 1);
            if ((quad + 1) * 4 * kBlock4 <= k) load_quad4_of<T>(x + row * x_stride, quad, group, next[r]);
            else load_block4_of<T>(x + row * x_stride, quad * 4 + group, k, next[r]);
        }
    };
    if ((int64_t)blockIdx.x < tiles && quads > 0) load(blockIdx.x, 0);
    for (int i = threadIdx.x; i < quads * columns * 4; i += kHeadThreads4) {
        const int b = i & 3, column = i / 4 % columns, quad = i / 4 / columns;
        const int64_t source = min(column, n - 1);
        *reinterpret_cast<v4i*>(s_w + (quad * columns + column) * 64 + ((b ^ (column & 3)) * 16)) =
            load_block4(w.values + source * w.values_stride, quad * 4 + b, k);
        if (b == 0)
            *reinterpret_cast<uint32_t*>(s_e + (quad * columns + column) * 4) =
                load_exponents4(w.exponents + source * w.exponents_stride, quad, blocks);
    }
    __syncthreads();
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        v4f acc[R][TN];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[r][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int quad = 0; quad < quads; ++quad) {
            v4i q[R];
            uint32_t e[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if ((quad + 1) * 4 * kBlock4 <= k) exchange_quad4<T>(next[r]);
                q[r] = quantize_block4<T>(next[r], e[r]);
            }
            if (quad + 1 < quads) load(t, quad + 1);
            else if (t + gridDim.x < tiles) load(t + gridDim.x, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if (j * 16 >= n) break;
                const int column = quad * columns + j * 16 + (lane & 15);
                const v4i v = *reinterpret_cast<const v4i*>(s_w + column * 64 + ((group ^ (lane & 3)) * 16));
                const uint32_t scale = s_e[column * 4 + group];
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r][j] = multiply4<0, 0>(v, q[r], acc[r][j], scale, e[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t m0 = (t * kHeadWaves4 + wave) * kRows + r * 16;
            wave_lds_sync();
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int col = j * 16 + group * 4;
                O* const to = s_out + (lane & 15) * pitch + col;
                if (col + 4 <= n) {
                    Vec<O, 4> y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y.v[i] = from_float<O>(acc[r][j][i]);
                    if (pitch % 4 == 0) {  // LDS takes whole accesses where they are aligned
                        *reinterpret_cast<Vec<O, 4>*>(to) = y;
                    } else if (pitch % 2 == 0) {
                        reinterpret_cast<Vec<O, 2>*>(to)[0] = {y.v[0], y.v[1]};
                        reinterpret_cast<Vec<O, 2>*>(to)[1] = {y.v[2], y.v[3]};
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) to[i] = y.v[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (col + i < n) to[i] = from_float<O>(acc[r][j][i]);
                }
            }
            wave_lds_sync();
            const int rows = (int)max(min(m - m0, (int64_t)16), (int64_t)0);
            struct __attribute__((packed, aligned(sizeof(O)))) Loose {
                v4i v;
            };
            const auto move = [](O* to, const O* from) {  // a vector, aligned in LDS
                Loose y;
                y.v = *reinterpret_cast<const v4i*>(from);
                __builtin_nontemporal_store(y.v, &reinterpret_cast<Loose*>(to)->v);
            };
            if (pitch == n) {  // one stretch
                const int size = rows * n;
                O* const to = out + m0 * out_stride;
                for (int i = lane * kOct; i + kOct <= size; i += 64 * kOct) move(to + i, s_out + i);
                const int last = size / kOct * kOct + lane;
                if (last < size) to[last] = s_out[last];
            } else {
                int row = first_row, piece = first_piece;
                for (; row < rows; row += 64 / across, piece += 64 % across) {
                    if (piece >= across) {
                        piece -= across;
                        if (++row >= rows) break;
                    }
                    const int col = piece * kOct;
                    O* const to = out + (m0 + row) * out_stride + col;
                    const O* const from = s_out + row * pitch + col;
                    if (col + kOct <= n) {
                        move(to, from);
                    } else {
                        for (int c = 0; col + c < n; ++c) to[c] = from[c];
                    }
                }
            }
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

constexpr int64_t kHeadMostColumns4 = 256;

enum class Linear4Way { kFew, kHead, kTiles };

int64_t head4_weight_bytes(int64_t n, int64_t k) { return ceil_div(n, 16) * 16 * ceil_div(ceil_div(k, kBlock4), 4) * 68; }

// Few rows while their bytes, which every workgroup quantises, are few beside the weight's share of one (n = 32768, k = 4096 in
// bf16: one row 14.3 us against 17.5 through the tiled product, 8 rows 17.5 either way; n = k = 8192 in float32: 2 rows 12.3 against
// 14.4, 4 rows 16.3 against 14.6; n = 4096, k = 2048: 16 rows 7.9 against 9.5), and no wave's sum is longer than 65536 k. Few
// columns while the weight fits a workgroup's LDS, with rows enough that each of the GPU's CUs has its share (100 columns, k = 700:
// 8000 rows 18.7 us against 12.8, 32000 24 against 25; 150 columns, k = 128: 3000 rows 9.2 against 9.4, 307200 40 against 75).
Linear4Way linear4_way(int64_t x_bytes, int64_t m, int64_t n, int64_t k) {
    if (m <= kFewRows4 && m * k * x_bytes <= (n <= 4096 ? 131072 : 65536) && k <= 4 * kSumMostBlocks * kBlock)
        return Linear4Way::kFew;
    if (n <= kHeadMostColumns4 && head4_weight_bytes(n, k) <= kHeadBytes4 && m >= 4096 * ceil_div(k, 4 * kBlock4))
        return Linear4Way::kHead;
    return Linear4Way::kTiles;
}

int64_t linear4_rows_bytes(int64_t m, int64_t k) {  // of the rows of x in blocks: values, then exponents
    const int64_t blocks = ceil_div(k, kBlock4);
    return ceil_div(m * (blocks * 16 + ceil_div(blocks, 4) * 4), 256) * 256;
}

template <typename T, typename O>
gsx_hip_status launch_few4(const T* x, int64_t x_stride, const BlockMatrix& w, int64_t m, int64_t n, int64_t k, O* out,
                           int64_t out_stride, hipStream_t stream) {
    // waves enough for the GPU: up to 8 of them over k, four at least
    const int64_t chunks = ceil_div(ceil_div(k, kBlock4), kChunk4), groups = ceil_div(n, 16);
    int64_t waves = 4;
    while (waves < kFewWaves4 && waves < chunks && groups * waves < 4096) waves *= 2;
    int64_t span = kFewBytes4 / (kChunk4 * 17) / m;
    if (span > chunks) span = chunks;
    const FewShape shape = {(int)span};
    const int64_t lds = waves * 1024 + m * (shape.values_pitch() + shape.exponents_pitch());
    hipLaunchKernelGGL((linear4_few_kernel<T, O>), dim3((unsigned)(groups < 1024 ? groups : 1024)), dim3((unsigned)waves * 64),
                       (unsigned)lds, stream, x, x_stride, w, (int)m, n, k, shape, out, out_stride);
    return fields_launched("4-bit linear launch");
}

template <typename T, typename O, int TN>
gsx_hip_status launch_head4(const T* x, int64_t x_stride, const BlockMatrix& w, int64_t m, int64_t n, int64_t k, O* out,
                            int64_t out_stride, hipStream_t stream) {
    const int64_t tiles = ceil_div(m, kHeadRows4<T, TN> * kHeadWaves4);
    const int64_t lds = head4_weight_bytes(n, k) + kHeadWaves4 * 16 * head4_pitch<O>(n, out_stride) * (int64_t)sizeof(O);
    const int64_t each = std::min<int64_t>(163840 / (lds + 256), 4), most = 256 * (each < 1 ? 1 : each);
    hipLaunchKernelGGL((linear4_head_kernel<T, O, TN>), dim3((unsigned)(tiles < most ? tiles : most)), dim3(kHeadThreads4),
                       (unsigned)lds, stream, x, x_stride, w, m, (int)n, k, out, out_stride);
    return fields_launched("4-bit linear launch");
}

}  // namespace

extern "C" {

size_t gsx_hip_linear4_temp_bytes(int64_t m, int64_t n, int64_t k) {
    if (!product_sizes(m, n, k) || m == 0 || n == 0) return 0;
    // whatever the rows' type is: it decides where few rows end
    if (linear4_way(4, m, n, k) != Linear4Way::kTiles && linear4_way(2, m, n, k) != Linear4Way::kTiles) return 0;
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
    const Linear4Way way = linear4_way(type_bytes(x_type), m, n, k);
    if (way == Linear4Way::kTiles) {
        if (k > 0 && (temp == nullptr || !aligned_to(temp, 16)))
            return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit linear: the workspace must be non-null and 16-byte aligned");
        if (w_values_stride >= kMostStride || w_exponents_stride >= kMostStride / 4)
            return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE,
                               "4-bit linear: a wide layer's value rows lie less than 2^28 bytes apart, its exponent rows 2^26");
        const int64_t blocks = ceil_div(k, kBlock4), words = ceil_div(blocks, 4) * 4;
        uint8_t* const values = static_cast<uint8_t*>(temp);
        uint8_t* const exponents = values + m * blocks * 16;
        const gsx_hip_status st =
            gsx_hip_blocks4_quantize(x, x_type, m, k, x_stride, values, blocks * 16, exponents, words, stream);
        if (st != GSX_HIP_SUCCESS) return st;
        return gsx_hip_blocks4_matmul(values, blocks * 16, exponents, words, w_values, w_values_stride, w_exponents,
                                      w_exponents_stride, m, n, k, out, out_type, out_stride,
                                      values + linear4_rows_bytes(m, k), stream);
    }
    const BlockMatrix w = {w_values, w_exponents, w_values_stride, w_exponents_stride};
    return with_type(x_type, [&](auto tx) {
        return with_type(out_type, [&](auto to) {
            using T = decltype(tx);
            using O = decltype(to);
            const T* const from = static_cast<const T*>(x);
            O* const result = static_cast<O*>(out);
            if (way == Linear4Way::kFew) return launch_few4<T, O>(from, x_stride, w, m, n, k, result, out_stride, stream);
            if (n <= 64) return launch_head4<T, O, 4>(from, x_stride, w, m, n, k, result, out_stride, stream);
            if (n <= 160) return launch_head4<T, O, 10>(from, x_stride, w, m, n, k, result, out_stride, stream);
            return launch_head4<T, O, 16>(from, x_stride, w, m, n, k, result, out_stride, stream);
        });
    });
}

}  // extern "C"

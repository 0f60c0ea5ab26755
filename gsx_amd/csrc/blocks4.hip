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

#include <type_traits>

#include "blocks4.hpp"

namespace gsx_amd {

constexpr int kQuant4Threads = 256;
constexpr int kQuant4Unroll = 4;

// Four lanes per block, eight values a lane, kQuant4Unroll blocks one after the other: their loads are issued together. Bound by
// memory: 8192 x 8192 in bf16 26 to 32 us in a loop (5.3 to 6.5 TB/s).
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

// 16 bytes of the result a thread and store, so that a wave's stores follow one another without a gap, kExpand4Unroll of them 256
// threads apart. They pass the caches by. Bound by memory: 8192 x 8192 to float32 44 us
// (7 TB/s), 66 with 32 bytes a thread in two stores through them.
constexpr int kExpand4Unroll = 4;
template <typename O>
__global__ __launch_bounds__(kQuant4Threads) void expand4_kernel(const uint8_t* __restrict__ values, int64_t values_stride,
                                                                 const uint8_t* __restrict__ exponents,
                                                                 int64_t exponents_stride, int64_t rows, int64_t cols,
                                                                 O* __restrict__ out, int64_t out_stride) {
    constexpr int kEach = 16 / (int)sizeof(O);
    struct __attribute__((packed, aligned(sizeof(O)))) Loose {
        v4i v;
    };
    struct Piece {
        O v[kEach];
    };
    const int64_t pieces = ceil_div(cols, kEach), total = rows * pieces;
    const int64_t whole = kQuant4Threads / pieces, rest = kQuant4Threads % pieces;  // 256 pieces on
    for (int64_t b = blockIdx.x; b * (kQuant4Threads * kExpand4Unroll) < total; b += gridDim.x) {
        const int64_t i = b * (kQuant4Threads * kExpand4Unroll) + threadIdx.x;
        int64_t r = total <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)pieces) : i / pieces, piece = i - r * pieces;
        const auto on = [&] {
            r += whole;
            piece += rest;
            if (piece >= pieces) {
                piece -= pieces;
                ++r;
            }
        };
        int64_t row[kExpand4Unroll], at[kExpand4Unroll];
        uint32_t q[kExpand4Unroll], e[kExpand4Unroll];
#pragma unroll
        for (int u = 0; u < kExpand4Unroll; ++u) {
            row[u] = r;
            at[u] = piece * kEach;
            q[u] = e[u] = 0;
            if (r < rows) {
                const uint8_t* const from = values + r * values_stride + at[u] / 2;
                if constexpr (kEach == 8) q[u] = *reinterpret_cast<const uint32_t*>(from);
                else q[u] = *reinterpret_cast<const uint16_t*>(from);
                e[u] = exponents[r * exponents_stride + at[u] / kBlock4];
            }
            on();
        }
#pragma unroll
        for (int u = 0; u < kExpand4Unroll; ++u) {
            if (row[u] >= rows) break;
            const float scale = block4_scale(e[u]);
            const v2f x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], 1.0f, 0),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], 1.0f, 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], 1.0f, 2),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], 1.0f, 3)};
            Piece y;
#pragma unroll
            for (int j = 0; j < kEach; ++j) y.v[j] = from_float<O>(x[j / 2][j % 2] * scale);
            O* const to = out + row[u] * out_stride + at[u];
            if (at[u] + kEach <= cols) {
                __builtin_nontemporal_store(__builtin_bit_cast(v4i, y), &reinterpret_cast<Loose*>(to)->v);
            } else {
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (at[u] + j < cols) to[j] = y.v[j];
            }
        }
    }
}

// ---- product ------------------------------------------------------------------------------------------------------------
//
// A workgroup of WM x WN waves forms a tile of c: BM rows (of a) by BN columns (rows of b), a wave TM x TN times 16 x 16 of it.
// Eight blocks, 256 k, of both operands' tiles lie in LDS, two such steps at a time: while one is multiplied the next is on its way
// there, straight from memory. A row is eight chunks of 16 bytes, one block each; chunk c lies at place c ^ swizzle(row), and a lane
// of group g = lane / 16 reads chunks g and g + 4: no two lanes of a read of values meet in a bank. A row's exponents of two steps lie
// behind one another, as in memory, 16 bytes a row: those of rows 16 apart share a bank, which b's reads for 16-bit results meet
// (conflicts in 13% of the cycles of 8192^3 to bf16; 5% in a product to float32, whose reads take 16 rows in a row).
//
// The matrix instructions take b as their first operand: a lane then holds four consecutive columns of one row of c. Which
// row of b a lane brings for instruction j is chosen so that it has 16 bytes of columns together and that the four lanes of a row
// store 64 bytes in a piece: 32 columns by a pair of instructions in 16-bit types, 16 by one in float32.
//
// 8192^3 to bf16: 285 to 300 us by the card, 3.7 to 3.85 PFLOP/s, 471 before the loads of the next step were in flight beside the
// instructions, exponents came two steps at a time and rows left in pieces of 64 bytes. The matrix units are busy for 41% of the
// cycles; the waves spend 35% of their lives in waits and 36% waiting for issue. Every step waits for all of its loads, so that no
// more than one step of 256 k is on its way. Four rows of tiles read ahead instead of two, a higher priority for the instructions or 4
// waves of 128 x 128 made it no faster (0, 0 and -7%); shorter steps, more of them on their way, have not been tried.
constexpr int kStep4 = 8;  // blocks

template <typename O>
constexpr int kPair = sizeof(O) == 2 ? 2 : 1;  // instructions whose columns of a lane lie together
template <typename O>
__device__ constexpr int column4_of(int j, int r) {
    return j / kPair<O> * (16 * kPair<O>) + r / 4 * (4 * kPair<O>) + j % kPair<O> * 4 + r % 4;
}
template <typename O>
__device__ inline int swizzle4_b(int row) {
    return kPair<O> == 2 ? (row & 3) | (row >> 3 & 1) << 2 : row & 7;
}

// store_row4 for 16-bit rows that begin between two words: a lane's pieces go one column on, the column behind comes from the next
// lane of the row. Whole words cost less than the same vectors two bytes off: 29681 x 2261 x 22 64 us, the latter way 80.
template <int TN, typename S>
__device__ inline void store_shifted4(S* __restrict__ row, int64_t col, int64_t n, int lane, const v4f (&x)[TN]) {
    struct __attribute__((packed, aligned(4))) Piece {
        S v[8];
    };
    const int group = lane / 16;
    if (group == 0 && col < n) row[col] = from_float<S>(x[0][0]);
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
        const bool last = group == 3 && j + 2 >= TN;
        const float behind = __shfl(group == 0 && j + 2 < TN ? x[j + 2 < TN ? j + 2 : j][0] : x[j][0], (lane + 16) & 63, 64);
        const int64_t c = col + 16 * j + group * 8 + 1;
        Piece q;
#pragma unroll
        for (int i = 0; i < 7; ++i) q.v[i] = from_float<S>(x[j + (i + 1) / 4][(i + 1) % 4]);
        q.v[7] = from_float<S>(behind);
        if (c + 8 <= n && !last) {
            *reinterpret_cast<Piece*>(row + c) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < n && !(last && i == 7)) row[c + i] = q.v[i];
        }
    }
}

// A lane's 4 TN columns of a row of n, the first of them at `col` + 4 kPair<O> (lane / 16). A store has 64 bytes of 16 rows; 128 of 8
// rows, after an exchange between lanes, were slower (29681 x 2304 x 256 to bf16 53 us, 71), stores past the caches too (58).
template <typename O, int TN, typename S>
__device__ inline void store_row4(S* __restrict__ row, int64_t col, int64_t n, int lane, const v4f (&x)[TN]) {
    constexpr int kP = kPair<O>;
    if constexpr (sizeof(S) == 2) {
        if (reinterpret_cast<uintptr_t>(row + col) % 4 != 0) {
            store_shifted4<TN>(row, col, n, lane, x);
            return;
        }
    }
    struct __attribute__((packed, aligned(sizeof(S)))) Piece {
        S v[4 * kP];
    };
#pragma unroll
    for (int j = 0; j < TN; j += kP) {
        const int64_t c = col + 16 * j + lane / 16 * (4 * kP);
        if (c + 4 * kP <= n) {
            Piece q;
#pragma unroll
            for (int i = 0; i < 4 * kP; ++i) q.v[i] = from_float<S>(x[j + i / 4][i % 4]);
            *reinterpret_cast<Piece*>(row + c) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 4 * kP; ++i)
                if (c + i < n) row[c + i] = from_float<S>(x[j + i / 4][i % 4]);
        }
    }
}

// Where a wave's loads begin: of the values of a step a load brings eight rows, of the exponents of two steps 64.
template <int kLoads, int kExponentLoads>
struct StepLoads4 {
    const uint8_t *a, *b, *a_exponents, *b_exponents;  // the tile's rows
    uint32_t offset[kLoads];                           // in units of 16 bytes
    uint32_t exponent_offset[kExponentLoads];          // and of 4
};

// The chunk of a row that a lane of load u brings.
template <typename O, int BM, int kWaves>
__device__ __forceinline__ int chunk4_of(int u, int wave, int lane) {
    const int row = 8 * (u * kWaves + wave) + lane / 8;
    return (lane & 7) ^ (row < BM ? swizzle_a(row) : swizzle4_b<O>(row - BM));
}

// A step's values; of its chunks from `chunks` on (of a cut step, the last one) the last one before them is read again.
template <typename O, int kLoads, int kExponentLoads, int BM, int kWaves>
__device__ __forceinline__ void load_step4(uint8_t* __restrict__ to, const StepLoads4<kLoads, kExponentLoads>& from, int step,
                                           int chunks, int wave, int lane) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const uint8_t* const base = (8 * (u * kWaves + wave) < BM ? from.a : from.b) + (uint32_t)step * 128;
        uint32_t offset = from.offset[u];
        if (chunks < kStep4) offset -= (uint32_t)max(chunk4_of<O, BM, kWaves>(u, wave, lane) - (chunks - 1), 0);
        __builtin_amdgcn_global_load_lds((GlobalPtr)(base + (uint64_t)offset * 16), (LdsPtr)(to + (u * kWaves + wave) * 1024), 16,
                                         0, 0);
    }
}

template <int kLoads, int kExponentLoads, int kRows, int BM, int kWaves>
__device__ __forceinline__ void load_exponents4(uint8_t* __restrict__ to, const StepLoads4<kLoads, kExponentLoads>& from, int pair,
                                                int wave) {
#pragma unroll
    for (int u = 0; u < kExponentLoads; ++u) {
        const int row = (u * kWaves + wave) * 64;
        if (row >= kRows) continue;
        const uint8_t* const base = (row < BM ? from.a_exponents : from.b_exponents) + (uint32_t)pair * 16;
        __builtin_amdgcn_global_load_lds((GlobalPtr)(base + (uint64_t)from.exponent_offset[u] * 4),
                                         (LdsPtr)(to + (u * kWaves + wave) * 1024), 16, 0, 0);
    }
}

// The lane's places in a step: chunk lane / 16 of its first row of each operand (the one four further is 64 bytes away, up or
// down), and its exponent there.
struct StepPlaces4 {
    int a, b, e_a, e_b;
};

// What a cut step's operands are masked with: of the lane's two chunks the bits that are there, and whether any are.
struct Cut4 {
    v4i keep[2];
    bool some[2];
};
__device__ inline Cut4 cut4_of(int64_t left, int group) {  // values that are left of the step
    Cut4 cut;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int mine = (int)max(min(left - (group + 4 * half) * kBlock4, (int64_t)kBlock4), (int64_t)0);
        cut.some[half] = mine > 0;
#pragma unroll
        for (int d = 0; d < 4; ++d) cut.keep[half][d] = (int)(0xffffffffull >> (32 - max(min(4 * (mine - 8 * d), 32), 0)));
    }
    return cut;
}

// One step: the loads of the next one are begun, then this one, which they do not touch, is multiplied. __restrict__ says so to the
// compiler, which otherwise waits for the loads before it reads LDS. What the instructions of two rows of tiles need is read ahead.
// kCut: this is the last step and cut. Zeros of a times anything of b are 0, but for a scale that is NaN.
template <bool kCut, typename O, int TM, int TN, int kRows, int BM, int kWaves, int kLoads, int kExponentLoads>
__device__ __forceinline__ void product4_step(const uint8_t* __restrict__ now, const uint8_t* __restrict__ exponents,
                                              uint8_t* __restrict__ next, uint8_t* __restrict__ next_exponents, int load_chunks,
                                              bool load_exponents, const StepLoads4<kLoads, kExponentLoads>& from, int step,
                                              int wave, int lane, StepPlaces4 at, const Cut4& cut, v4f (&acc)[TM][TN]) {
    if (load_chunks > 0) load_step4<O, kLoads, kExponentLoads, BM, kWaves>(next, from, step, load_chunks, wave, lane);
    if (load_exponents) load_exponents4<kLoads, kExponentLoads, kRows, BM, kWaves>(next_exponents, from, step / 2, wave);
    constexpr int kAhead = 3;
    v4i va[kAhead], vb[2][TN];
    uint32_t scale_a[kAhead], scale_b[2][TN];
    const auto read_a = [&](int n) {  // of both halves' rows of tiles
        const int i = n % TM, half = n / TM;
        va[n % kAhead] = *reinterpret_cast<const v4i*>(now + (at.a ^ (half * 64)) + i * (16 * 128));
        scale_a[n % kAhead] = exponents[at.e_a + half * 4 + i * (16 * 16)];
        if constexpr (kCut) {
            va[n % kAhead] &= cut.keep[half];
            if (!cut.some[half]) scale_a[n % kAhead] = 127;
        }
    };
    const auto read_b = [&](int half, int j) {
        const int row = column4_of<O>(j, 0);
        vb[half][j] = *reinterpret_cast<const v4i*>(now + (at.b ^ (half * 64)) + row * 128);
        scale_b[half][j] = exponents[at.e_b + half * 4 + row * 16];
        if constexpr (kCut) {
            if (!cut.some[half]) scale_b[half][j] = 127;
        }
    };
#pragma unroll
    for (int j = 0; j < TN; ++j) read_b(0, j);
#pragma unroll
    for (int n = 0; n < kAhead - 1; ++n) read_a(n);
#pragma unroll
    for (int n = 0; n < 2 * TM; ++n) {
        const int i = n % TM, half = n / TM;
        if (n + kAhead - 1 < 2 * TM) read_a(n + kAhead - 1);
        if (n < TN) read_b(1, n);
        __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of the instructions
#pragma unroll
        for (int j = 0; j < TN; ++j)
            acc[i][j] = multiply4<0, 0>(vb[half][j], va[n % kAhead], acc[i][j], scale_b[half][j], scale_a[n % kAhead]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <typename O, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void product4_kernel(BlockMatrix a, BlockMatrix b, int64_t m, int64_t n, int64_t k,
                                                                int64_t tiles_m, int64_t tiles_n, int64_t splits,
                                                                O* __restrict__ out, int64_t out_stride,
                                                                float* __restrict__ partial) {
    constexpr int kThreads = 64 * WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
    constexpr int kRows = BM + BN, kLoads = kRows * 8 / kThreads, kWaves = WM * WN;
    constexpr int kExponentLoads = (kRows / 64 + kWaves - 1) / kWaves;
    static_assert(kRows * 8 % kThreads == 0 && BM % (8 * kWaves) == 0 && BM % 64 == 0, "whole loads, each of one operand");
    static_assert(TN <= TM && TN % 2 == 0, "b's second half is read beside the first one's instructions");
    __shared__ __attribute__((aligned(1024))) uint8_t s_values[2][kRows * 128];
    __shared__ __attribute__((aligned(1024))) uint8_t s_exponents[2][kRows * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN, wn = wave % WN, group = lane / 16;
    const int blocks = (int)ceil_div(k, kBlock4), steps = (int)ceil_div(blocks, kStep4);
    const int64_t total = tiles_m * tiles_n * splits;
    const int row_a = wm * 16 * TM + (lane & 15), row_b = wn * 16 * TN + column4_of<O>(0, lane & 15);
    const StepPlaces4 even = {row_a * 128 + ((group ^ swizzle_a(row_a)) * 16),
                              (BM + row_b) * 128 + ((group ^ swizzle4_b<O>(row_b)) * 16), row_a * 16 + group,
                              (BM + row_b) * 16 + group};
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const ProductTile tile = product_tile(t, total, tiles_m, tiles_n, BM, BN, steps, splits);
        const int first = (int)tile.first, count = (int)(tile.last - tile.first);
        // Load u of a wave: eight rows (lane / 8) from row 8 (u kWaves + wave) on, a's rows before b's. Rows past the last one
        // repeat it; what they give is not stored.
        const int most_a = (int)min(m - 1 - tile.m0, (int64_t)BM), most_b = (int)min(n - 1 - tile.n0, (int64_t)BN);
        const uint32_t a_step = (uint32_t)(a.values_stride / 16), b_step = (uint32_t)(b.values_stride / 16);
        const uint32_t a_words = (uint32_t)(a.exponents_stride / 4), b_words = (uint32_t)(b.exponents_stride / 4);
        StepLoads4<kLoads, kExponentLoads> from;
        from.a = a.values + tile.m0 * a.values_stride;
        from.b = b.values + tile.n0 * b.values_stride;
        from.a_exponents = a.exponents + tile.m0 * a.exponents_stride;
        from.b_exponents = b.exponents + tile.n0 * b.exponents_stride;
        const auto exponent_row = [&](int row) {
            return row < BM ? min(row, most_a) * a_words : min(row - BM, most_b) * b_words;
        };
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int row = 8 * (u * kWaves + wave) + lane / 8;
            from.offset[u] = (row < BM ? min(row, most_a) * a_step : min(row - BM, most_b) * b_step) +
                             (uint32_t)chunk4_of<O, BM, kWaves>(u, wave, lane);
        }
#pragma unroll
        for (int u = 0; u < kExponentLoads; ++u)
            from.exponent_offset[u] = exponent_row(min((u * kWaves + wave) * 64, kRows - 64) + lane);
        // exponents of a pair of steps that is cut: through registers, a word a thread
        const auto stage_exponents = [&](int pair, uint8_t* to) {
            const int word = pair * 4 + (threadIdx.x & 3), at = min(word, (blocks - 1) / 4);
            const int left = max(min(blocks - 4 * word, 4), 0);
            const uint32_t keep = (uint32_t)((1ull << (8 * left)) - 1);
#pragma unroll 2
            for (int i = threadIdx.x; i < 4 * kRows; i += kThreads) {
                const uint32_t* const p =
                    reinterpret_cast<const uint32_t*>(i / 4 < BM ? from.a_exponents : from.b_exponents) + exponent_row(i / 4);
                reinterpret_cast<uint32_t*>(to)[i] = (p[at] & keep) | (0x7f7f7f7fu & ~keep);
            }
        };
        const auto chunks_of = [&](int step) { return min(blocks - step * kStep4, kStep4); };
        const auto whole_pair = [&](int step) { return (step / 2 * 2 + 2) * kStep4 <= blocks; };
        v4f acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        int held = 0;  // the buffer of this step's exponents
        if (count > 0) {
            load_step4<O, kLoads, kExponentLoads, BM, kWaves>(s_values[0], from, first, chunks_of(first), wave, lane);
            if (whole_pair(first))
                load_exponents4<kLoads, kExponentLoads, kRows, BM, kWaves>(s_exponents[0], from, first / 2, wave);
            else
                stage_exponents(first / 2, s_exponents[0]);
        }
        const auto multiply = [&](auto cut_step, int i) {
            // This step is in LDS (the barrier does not wait for loads that go there), the one before it has been read.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            constexpr bool kCut = decltype(cut_step)::value;
            const int step = first + i, next = step + 1;
            const bool more = !kCut && i + 1 < count, turns = more && next % 2 == 0, cut_pair = turns && !whole_pair(next);
            if (cut_pair) stage_exponents(next / 2, s_exponents[held ^ 1]);
            const StepPlaces4 places = {even.a, even.b, even.e_a + (step & 1) * 8, even.e_b + (step & 1) * 8};
            const Cut4 cut = kCut ? cut4_of(k - (int64_t)step * kStep4 * kBlock4, group) : Cut4{};
            product4_step<kCut, O, TM, TN, kRows, BM, kWaves, kLoads, kExponentLoads>(
                s_values[i & 1], s_exponents[held], s_values[(i + 1) & 1], s_exponents[held ^ 1], more ? chunks_of(next) : 0,
                turns && !cut_pair, from, next, wave, lane, places, cut, acc);
            if (turns) held ^= 1;
        };
        const bool cut = count > 0 && (int64_t)(first + count) * kStep4 * kBlock4 > k;
        for (int i = 0; i < count - (cut ? 1 : 0); ++i) multiply(std::false_type(), i);
        if (cut) multiply(std::true_type(), count - 1);
        __syncthreads();  // the next tile's first step goes where this one's last was read
        const int64_t col = tile.n0 + wn * 16 * TN;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int64_t row = tile.m0 + wm * 16 * TM + i * 16 + (lane & 15);
            if (row >= m) continue;
            if (splits == 1) {
                store_row4<O, TN>(out + row * out_stride, col, n, lane, acc[i]);
            } else {
                store_row4<O, TN>(partial + (tile.split * m + row) * n, col, n, lane, acc[i]);
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

// Tiles and splits of a product by its sizes alone: what is estimated to take the least time. A round of tiles (256 or 192 wide one
// to a CU, 128 two, 64 four) takes a fixed time, most of it the stores, and one a step of 256 k; in tenths of a microsecond, from
// 8192 x 8192 x 256 to 8192: 8192 with tiles of 64 498 us, 128 346, 192 391, 256 285; 256 63, 50, 59 and 46. Narrow tiles pay where
// wide ones leave CUs without work (493 x 7309 x 1940: 17 us, 27, 29 and 35) or fill the last round badly. What fills less than
// half a round may also be split over k, two steps or more to a part; the parts' sums are then written, read and joined.
struct Product4Plan {
    int edge;
    int64_t tiles_m, tiles_n, splits;
    int64_t temp_bytes;
};

constexpr int64_t kSum4MostSteps = kSumMostBlocks * kBlock / (kStep4 * kBlock4);  // 65536 k, after which a float sum starts anew

Product4Plan product4_plan(int64_t m, int64_t n, int64_t k) {
    struct Tiles {
        int edge;
        int64_t slots, round, step;
    };
    constexpr Tiles kTiles[] = {{256, 256, 90, 19}, {192, 256, 60, 15}, {128, 512, 50, 12}, {64, 1024, 25, 9}};
    const int64_t steps = ceil_div(k, kStep4 * kBlock4), least = k > 0 ? ceil_div(steps, kSum4MostSteps) : 1;
    Product4Plan p = {};
    int64_t best = INT64_MAX;
    for (const Tiles& t : kTiles) {
        if (t.edge > 64 && (m <= 64 || n <= 64)) continue;
        const int64_t count = ceil_div(m, t.edge) * ceil_div(n, t.edge);
        int64_t most = count < t.slots / 2 ? t.slots / count : 1;  // one round of workgroups
        if (most > steps / 2) most = steps / 2;
        for (const int64_t splits : {least, most / 2, most}) {
            if (splits < least) continue;
            int64_t cost = ceil_div(count * splits, t.slots) * (t.round + t.step * ceil_div(steps, splits));
            if (splits > 1) cost += 40 + splits * (m * n / 50000);
            if (cost >= best) continue;
            best = cost;
            p.edge = t.edge;
            p.splits = splits;
        }
    }
    p.tiles_m = ceil_div(m, p.edge);
    p.tiles_n = ceil_div(n, p.edge);
    p.temp_bytes = p.splits > 1 ? p.splits * m * n * 4 : 0;
    return p;
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
        const int64_t pieces = rows * ceil_div(cols, 16 / (int64_t)sizeof(O));
        hipLaunchKernelGGL((expand4_kernel<O>), dim3(blocks_grid(ceil_div(pieces, kQuant4Threads * kExpand4Unroll))),
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
    if (a_values_stride >= kMostStride || b_values_stride >= kMostStride || a_exponents_stride >= kMostStride / 4 ||
        b_exponents_stride >= kMostStride / 4)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE,
                           "4-bit blocks: a product's value rows lie less than 2^28 bytes apart, its exponent rows 2^26");
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
        else if (plan.edge == 192) go(product4_kernel<O, 6, 4, 2, 3>, 384);
        else if (plan.edge == 128) go(product4_kernel<O, 4, 4, 2, 2>, 256);
        else go(product4_kernel<O, 2, 2, 2, 2>, 256);
        if (plan.splits > 1) launch_join(partial, m, n, plan.splits, to, out_stride, stream);
        return fields_launched("4-bit blocks matmul launch");
    });
}

}  // extern "C"

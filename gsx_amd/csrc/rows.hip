// rows.hip - rows of a table looked up by id and scaled, and the table's gradient.
//
//   out[i, :] = s * table[id_i, :]            (an id outside the table: zeros)
//   G[v, :]   = s * sum over i with id_i = v of g[i, :]
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.hpp"
#include "fields.hpp"

namespace gsx_amd {

constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;
constexpr int kRowTile = kRowThreads * kRowUnroll;  // vectors of V elements a workgroup copies at a time
constexpr int64_t kRowMostBlocks = 1 << 20;

// V elements at any element's address: rows of odd widths and strides move in wide vectors too (150000 x 385 looked up: 54 us, one
// element at a time 105).
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T v[V];
};

// What these kernels write is much, written once and read by a later launch: it passes the caches by and leaves what is read in
// them (1M rows of 64 looked up: 44 us against 60; the gradient of 65536 x 2048: 104 against 158).
template <typename O, int V>
__device__ inline void store_past_caches(O* p, const Span<O, V>& y) {
    if constexpr (V * sizeof(O) == 16) {
        typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(4)));
        typedef uint32_t Words2 __attribute__((ext_vector_type(4), aligned(2)));
        using Words = std::conditional_t<sizeof(O) == 4, Words4, Words2>;
        __builtin_nontemporal_store(__builtin_bit_cast(Words, y), reinterpret_cast<Words*>(p));
    } else {
        *reinterpret_cast<Span<O, V>*>(p) = y;
    }
}

// Column at which vector `vec` of a row begins. A last vector that would end behind the row is moved back into it: its first
// columns are the vector's before too, and both form the same values for them.
template <int V>
__device__ inline int64_t column_at(int64_t vec, int64_t width) {
    return min(vec * V, width - V);
}

// A tile is `tile_rows` whole rows of `vecs` vectors, or (vecs > kRowTile) a part of one row. Every id, then every row vector
// of a thread is loaded before the first store. The stores bound it: 1M rows of 64 float32 from a table that the caches hold, 256
// MB written in 44 us (5.9 TB/s; a fill reaches 6.9). One row of 4096 bf16: 2.4 us.
template <typename T, typename O, int V>
__global__ __launch_bounds__(kRowThreads) void lookup_kernel(const T* __restrict__ table, int64_t table_rows,
                                                             int64_t table_stride, const int32_t* __restrict__ ids,
                                                             int64_t count, int64_t width, int tile_rows, int64_t parts,
                                                             int64_t tiles, float scale, O* __restrict__ out,
                                                             int64_t out_stride, int* __restrict__ out_of_range) {
    const int64_t vecs = ceil_div(width, V);
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row0 = tile / parts * tile_rows;
        const int64_t col0 = tile % parts * kRowTile;
        const uint32_t cols = (uint32_t)min(vecs - col0, (int64_t)kRowTile);
        const uint32_t work = (uint32_t)min((int64_t)tile_rows, count - row0) * cols;
        int32_t id[kRowUnroll];
        int64_t row[kRowUnroll], col[kRowUnroll];
        Span<T, V> x[kRowUnroll];
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            const uint32_t e = threadIdx.x + u * kRowThreads;
            row[u] = row0 + e / cols;
            col[u] = column_at<V>(col0 + e % cols, width);
            id[u] = e < work ? ids[row[u]] : -1;
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            if (id[u] >= 0 && id[u] < table_rows)
                x[u] = *reinterpret_cast<const Span<T, V>*>(table + (int64_t)id[u] * table_stride + col[u]);
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            if (threadIdx.x + u * kRowThreads >= work) continue;
            const bool fits = id[u] >= 0 && id[u] < table_rows;
            if (id[u] >= table_rows && out_of_range != nullptr) *out_of_range = 1;
            Span<O, V> y;
#pragma unroll
            for (int k = 0; k < V; ++k) y.v[k] = from_float<O>(fits ? to_float(x[u].v[k]) * scale : 0.0f);
            store_past_caches<O, V>(out + row[u] * out_stride + col[u], y);
        }
    }
}

// ---- gradient -----------------------------------------------------------------------------------------------------------
//
// Few ids: one wave per table row and some vectors of V columns reads all ids, 64 at a time, and adds the rows of its id (77 ids,
// 1001 rows of 385: 3.6 us, near a launch's least). It hardly reads, so its stores stay in the caches as far as they fit (4 ids,
// 56074 rows of 900: 27 us against 47, 100000 of 1024: 72 either way).
//
// Many: the ids are sorted with their positions as values (ids outside the table as table_rows, behind all others), so each
// table row owns a run of positions. Runs of up to kRunPart rows are summed by one group of lanes each; longer ones in parts of
// kRunPart sorted positions, whose sums a last launch joins. Every sum has a fixed order, so results repeat bit for bit, and
// the most frequent id's run is spread over as many workgroups as it has parts. Memory bounds the sums (16384 bf16 rows of 2048
// into 65536: 101 us for 604 MB, 6 TB/s; 1M float32 rows of 64 into 8192: 57 us for 258 MB, 4.5 TB/s), the latency of some
// eight small launches what comes before and behind (34 and 50 us in these cases).

constexpr int kRunPart = 128;

template <typename T, int V>
__device__ inline void add_span(float (&sum)[V], const Span<T, V>& x) {
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] += to_float(x.v[k]);
}

// Vector `vec` of a row of the result, past the caches or not.
template <int V, bool kPast>
__device__ inline void store_row(float* row, int64_t vec, int64_t width, const float (&sum)[V], float scale, bool accumulate) {
    const int64_t col = column_at<V>(vec, width);
    float* const p = row + col;
    if (accumulate && col != vec * V) {  // the vector before adds to the columns they share
        for (int k = (int)(vec * V - col); k < V; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i == k) p[k] += sum[i] * scale;
        return;
    }
    Span<float, V> y;
#pragma unroll
    for (int k = 0; k < V; ++k) y.v[k] = sum[k] * scale;
    if (accumulate) {
        const Span<float, V> old = *reinterpret_cast<const Span<float, V>*>(p);
#pragma unroll
        for (int k = 0; k < V; ++k) y.v[k] += old.v[k];
    }
    if constexpr (kPast) store_past_caches<float, V>(p, y);
    else *reinterpret_cast<Span<float, V>*>(p) = y;
}

// kTiles times 64 vectors of a row a wave, or (kSplit > 1) 64 vectors a workgroup, whose waves take every kSplit-th 64 ids each.
template <typename T, int V, int kTiles, int kSplit>
__global__ __launch_bounds__(kRowThreads) void lookup_scan_kernel(const T* __restrict__ grad, int64_t grad_stride,
                                                                  const int32_t* __restrict__ ids, int64_t count,
                                                                  float scale, float* __restrict__ out,
                                                                  int64_t table_rows, int64_t out_stride, int64_t width,
                                                                  int accumulate) {
    static_assert(kSplit == 1 || (kSplit == kRowThreads / 64 && kTiles == 1), "a workgroup's waves share one row");
    constexpr int kAhead = 8 / kTiles;  // rows whose loads are in flight together
    __shared__ float s_sum[kSplit][kSplit > 1 ? 64 * V : 1];
    __shared__ int s_any;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int64_t vecs = ceil_div(width, V), parts = ceil_div(vecs, 64 * kTiles);
    const int64_t works = table_rows * parts, per_block = kRowThreads / 64 / kSplit;
    for (int64_t w = blockIdx.x * per_block + (kSplit > 1 ? 0 : wave); w < works; w += gridDim.x * per_block) {
        const int64_t v = w / parts;
        const int64_t first = w % parts * 64 * kTiles + lane;
        float sum[kTiles][V] = {};
        bool any = false;
        if constexpr (kSplit > 1) {
            if (threadIdx.x == 0) s_any = 0;
            __syncthreads();
        }
        for (int64_t at = kSplit > 1 ? 64 * wave : 0; at < count; at += 64 * kSplit) {
            const int32_t id = at + lane < count ? ids[at + lane] : -1;
            uint64_t mine = __builtin_amdgcn_ballot_w64(id == v);
            while (mine != 0) {
                any = true;
                Span<T, V> x[kAhead][kTiles];
                bool some[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    some[u] = mine != 0;
                    if (!some[u]) continue;
                    const T* const row = grad + (at + __builtin_ctzll(mine)) * grad_stride;
                    mine &= mine - 1;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        x[u][t] = *reinterpret_cast<const Span<T, V>*>(row + column_at<V>(min(first + 64 * t, vecs - 1), width));
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (some[u])
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) add_span<T, V>(sum[t], x[u][t]);
            }
        }
        if constexpr (kSplit > 1) {
            if (any && lane == 0) s_any = 1;
#pragma unroll
            for (int k = 0; k < V; ++k) s_sum[wave][k * 64 + lane] = sum[0][k];
            __syncthreads();
            any = s_any != 0;
            if (wave == 0)
                for (int i = 1; i < kSplit; ++i)
#pragma unroll
                    for (int k = 0; k < V; ++k) sum[0][k] += s_sum[i][k * 64 + lane];
            __syncthreads();
            if (wave != 0) continue;
        }
        if (!any && accumulate != 0) continue;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
            if (first + 64 * t < vecs)
                store_row<V, false>(out + v * out_stride, first + 64 * t, width, sum[t], scale, accumulate != 0);
    }
}

template <typename KeyT>
__global__ __launch_bounds__(kRowThreads) void lookup_keys_kernel(const int32_t* __restrict__ ids, int64_t count,
                                                                  int32_t table_rows, KeyT* __restrict__ keys) {
    for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kRowThreads) {
        const int32_t id = ids[i];
        keys[i] = (KeyT)(id >= 0 && id < table_rows ? id : table_rows);
    }
}

// starts[v] = the number of sorted keys below v, for v in [0, table_rows]: a binary search each, 5 to 7 us of latency.
template <typename KeyT>
__global__ __launch_bounds__(kRowThreads) void lookup_starts_kernel(const KeyT* __restrict__ keys, int64_t count,
                                                                    int64_t table_rows, uint32_t* __restrict__ starts) {
    for (int64_t v = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; v <= table_rows;
         v += (int64_t)gridDim.x * kRowThreads) {
        int64_t lo = 0, hi = count;
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if ((int64_t)keys[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        starts[v] = (uint32_t)lo;
    }
}

// Sum over sorted positions [begin, end), `step` apart from `begin` on, of the rows' vector at `col`.
template <typename T, int V>
__device__ inline void sum_run(float (&sum)[V], const T* __restrict__ grad, int64_t grad_stride,
                               const uint32_t* __restrict__ order, uint32_t begin, uint32_t end, uint32_t step,
                               int64_t col) {
    constexpr int kAhead = 4;  // rows whose loads are in flight together
    int64_t p = begin;
    for (; p + (kAhead - 1) * (int64_t)step < end; p += kAhead * (int64_t)step) {
        Span<T, V> x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            x[u] = *reinterpret_cast<const Span<T, V>*>(grad + (int64_t)order[p + u * (int64_t)step] * grad_stride + col);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) add_span<T, V>(sum, x[u]);
    }
    for (; p < end; p += step)
        add_span<T, V>(sum, *reinterpret_cast<const Span<T, V>*>(grad + (int64_t)order[p] * grad_stride + col));
}

// A group of `lanes` (a power of two, at most 64) lanes per table row and kTiles times `lanes` vectors of it. The loads of kAhead
// rows in all tiles are issued together; past the run's end the last row is loaded again and not added.
template <typename T, int V, int kTiles>
__device__ inline void sum_short_runs(const T* __restrict__ grad, int64_t grad_stride, const uint32_t* __restrict__ order,
                                      const uint32_t* __restrict__ starts, float scale, float* __restrict__ out,
                                      int64_t table_rows, int64_t out_stride, int64_t width, int lanes, int accumulate,
                                      int64_t block, int64_t blocks) {
    constexpr int kAhead = 8 / kTiles;
    const int64_t vecs = ceil_div(width, V);
    const int sub = threadIdx.x & (lanes - 1);
    const int64_t parts = ceil_div(vecs, (int64_t)lanes * kTiles);
    const int64_t groups = table_rows * parts, per_block = kRowThreads / lanes;
    for (int64_t g = block * per_block + threadIdx.x / lanes; g < groups; g += blocks * per_block) {
        const int64_t v = g / parts;
        const uint32_t begin = starts[v], end = starts[v + 1];
        if (end - begin > (uint32_t)kRunPart || (accumulate != 0 && begin == end)) continue;
        const int64_t first = g % parts * lanes * kTiles + sub;
        float sum[kTiles][V] = {};
        for (int64_t p = begin; p < end; p += kAhead) {
            Span<T, V> x[kAhead][kTiles];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const T* const row = grad + (int64_t)order[min(p + u, (int64_t)end - 1)] * grad_stride;
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    x[u][t] = *reinterpret_cast<const Span<T, V>*>(row + column_at<V>(min(first + t * lanes, vecs - 1), width));
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const bool some = p + u < end;  // a zero is added where there is no row: a sum is never -0
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int k = 0; k < V; ++k) sum[t][k] += some ? to_float(x[u][t].v[k]) : 0.0f;
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int64_t vec = first + t * lanes;
            if (vec < vecs) store_row<V, true>(out + v * out_stride, vec, width, sum[t], scale, accumulate != 0);
        }
    }
}

// Sorted positions [c kRunPart, (c + 1) kRunPart) cross at most two long runs, that of the first key (its sum goes to slot 0)
// and that of the last key if it is another one (slot 1). One wave per part and 64 vectors; fewer vectors leave 64 / lanes
// groups, each of which takes every so manieth position.
template <typename T, int V, typename KeyT>
__device__ inline void sum_long_parts(const T* __restrict__ grad, int64_t grad_stride, const uint32_t* __restrict__ order,
                                      const KeyT* __restrict__ keys, const uint32_t* __restrict__ starts, int64_t count,
                                      int64_t table_rows, int64_t width, int lanes, float* __restrict__ partial, int64_t block,
                                      int64_t blocks) {
    const int64_t vecs = ceil_div(width, V);
    const int64_t tiles = ceil_div(vecs, lanes);
    const int64_t waves = ceil_div(count, kRunPart) * tiles;
    const int lane = threadIdx.x & 63;
    for (int64_t w = block * (kRowThreads / 64) + threadIdx.x / 64; w < waves;
         w += blocks * (kRowThreads / 64)) {
        const int64_t c = w / tiles;
        const int64_t vec = w % tiles * lanes + (lane & (lanes - 1));
        const int64_t first = c * kRunPart, last = min(first + kRunPart, count) - 1;
        const int64_t k0 = keys[first], k1 = keys[last];
#pragma unroll 1
        for (int slot = 0; slot < 2; ++slot) {
            const int64_t key = slot == 0 ? k0 : k1;
            if (key >= table_rows || (slot == 1 && k1 == k0)) continue;
            const uint32_t begin = starts[key], end = starts[key + 1];
            if (end - begin <= (uint32_t)kRunPart) continue;
            float sum[V] = {};
            const uint32_t from = (uint32_t)max((int64_t)begin, first), to = (uint32_t)min((int64_t)end, last + 1);
            if (vec < vecs)
                sum_run<T, V>(sum, grad, grad_stride, order, from + lane / lanes, to, 64 / lanes, column_at<V>(vec, width));
            for (int off = lanes; off < 64; off <<= 1) {
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] += __shfl_xor(sum[k], off, 64);
            }
            if (vec < vecs && lane < lanes) {
                Vec<float, V> y;
#pragma unroll
                for (int k = 0; k < V; ++k) y.v[k] = sum[k];
                *reinterpret_cast<Vec<float, V>*>(partial + ((2 * c + slot) * vecs + vec) * V) = y;
            }
        }
    }
}

// Both in one launch: the first `part_blocks` workgroups take the long runs' parts, the others the short runs.
template <typename T, int V, int kTiles, typename KeyT>
__global__ __launch_bounds__(kRowThreads) void lookup_runs_kernel(const T* __restrict__ grad, int64_t grad_stride,
                                                                  const uint32_t* __restrict__ order,
                                                                  const KeyT* __restrict__ keys,
                                                                  const uint32_t* __restrict__ starts, int64_t count,
                                                                  float scale, float* __restrict__ out, int64_t table_rows,
                                                                  int64_t out_stride, int64_t width, int lanes,
                                                                  int accumulate, float* __restrict__ partial,
                                                                  int64_t part_blocks) {
    if ((int64_t)blockIdx.x < part_blocks) {
        sum_long_parts<T, V, KeyT>(grad, grad_stride, order, keys, starts, count, table_rows, width, lanes, partial, blockIdx.x,
                                   part_blocks);
    } else {
        sum_short_runs<T, V, kTiles>(grad, grad_stride, order, starts, scale, out, table_rows, out_stride, width, lanes,
                                     accumulate, blockIdx.x - part_blocks, gridDim.x - part_blocks);
    }
}

// The long run that begins among the positions of part c (at most one does: the last key's): its parts' sums in a fixed order,
// by the groups of a workgroup and then across them.
template <int V, typename KeyT>
__global__ __launch_bounds__(kRowThreads) void lookup_join_kernel(const KeyT* __restrict__ keys,
                                                                  const uint32_t* __restrict__ starts, int64_t count,
                                                                  int64_t table_rows, int64_t width, int lanes,
                                                                  const float* __restrict__ partial, float scale,
                                                                  float* __restrict__ out, int64_t out_stride,
                                                                  int accumulate) {
    __shared__ float s_sum[kRowThreads * V];
    const int64_t vecs = ceil_div(width, V);
    const int64_t tiles = ceil_div(vecs, lanes);
    const int64_t blocks = ceil_div(count, kRunPart) * tiles;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int64_t c = b / tiles;
        const int64_t first = c * kRunPart, last = min(first + kRunPart, count) - 1;
        const int64_t key = keys[last];
        if (key >= table_rows) continue;  // uniform, as the next
        const int64_t begin = starts[key], end = starts[key + 1];
        if (end - begin <= kRunPart || begin < first) continue;
        const int64_t vec = b % tiles * lanes + (threadIdx.x & (lanes - 1));
        const int groups = kRowThreads / lanes, group = threadIdx.x / lanes;
        float sum[V] = {};
        const int64_t final = (end - 1) / kRunPart;
        if (vec < vecs) {
            // a run that begins inside part c is that part's last key; in the later parts it is the first
            const float* const from = partial + vec * V;
            constexpr int kAhead = 8;
            for (int64_t p = c + group; p <= final; p += groups * kAhead) {
                Vec<float, V> x[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int64_t q = min(p + u * groups, final);
                    x[u] = *reinterpret_cast<const Vec<float, V>*>(from + (2 * q + (q == c && begin != first ? 1 : 0)) * vecs * V);
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (p + u * groups > final) continue;
#pragma unroll
                    for (int k = 0; k < V; ++k) sum[k] += x[u].v[k];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) s_sum[threadIdx.x * V + k] = sum[k];
        __syncthreads();
        if (group == 0 && vec < vecs) {
            for (int g = 1; g < groups; ++g)
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] += s_sum[(g * lanes + threadIdx.x) * V + k];
            store_row<V, true>(out + key * out_stride, vec, width, sum, scale, accumulate != 0);
        }
        __syncthreads();
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

template <typename T, typename O, int V>
gsx_hip_status launch_lookup(const void* table, int64_t table_rows, int64_t table_stride, const int32_t* ids,
                             int64_t count, int64_t width, float scale, void* out, int64_t out_stride, int* flag,
                             hipStream_t stream) {
    const int64_t vecs = ceil_div(width, V);
    const int tile_rows = vecs >= kRowTile ? 1 : (int)(kRowTile / vecs);
    const int64_t parts = ceil_div(vecs, kRowTile);
    const int64_t tiles = ceil_div(count, tile_rows) * parts;
    hipLaunchKernelGGL((lookup_kernel<T, O, V>), dim3((unsigned)(tiles < kRowMostBlocks ? tiles : kRowMostBlocks)),
                       dim3(kRowThreads), 0, stream, static_cast<const T*>(table), table_rows, table_stride, ids, count,
                       width, tile_rows, parts, tiles, scale, static_cast<O*>(out), out_stride, flag);
    return fields_launched("lookup launch");
}

// Few ids take the scan: one launch instead of ten, but every wave reads every id. More than 256 are shared by a workgroup's waves
// (2048 ids on 1000 rows 11 us against 36 by sorting, all of them on one row 35) while there are no more than some 16 000
// waves' rows (2048 ids on 16384 rows of 64 23 us against 35, on 65536 80
// against 42).
constexpr int64_t kScanSplit = 256;  // ids above which a workgroup's waves share them
constexpr int64_t kScanLong = 8192;  // waves that fill the GPU: from there on a wave takes 256 vectors of a row
bool takes_scan(int64_t count, int64_t table_rows, int64_t width) {
    return count <= kScanSplit || (count <= 2048 && table_rows * ceil_div(width, 256) <= 16384);
}

unsigned rows_grid(int64_t blocks) { return (unsigned)(blocks < kRowMostBlocks ? blocks : kRowMostBlocks); }

// Workspace of the sorted gradient: byte offsets of its arrays.
struct SortedIds {
    static bool narrow(int64_t table_rows) { return table_rows <= UINT16_MAX; }
    int64_t keys, keys_alt, keys_sorted, order_alt, order, sort, starts, partial, bytes;
    SortedIds(int64_t count, int64_t table_rows, int64_t width) {
        int64_t at = 0;
        const auto take = [&](int64_t size) {
            const int64_t here = at;
            at += ceil_div(size, 256) * 256;
            return here;
        };
        const int64_t key = narrow(table_rows) ? 2 : 4;
        keys = take(count * key);
        keys_alt = take(count * key);
        keys_sorted = take(count * key);
        order_alt = take(count * 4);
        order = take(count * 4);
        sort = take((int64_t)tile_sort_temp_bytes(count));
        starts = take((table_rows + 1) * 4);
        partial = take(ceil_div(count, kRunPart) * 2 * ceil_div(width, 4) * 16);
        bytes = at;
    }
};

template <typename T, int V, typename KeyT>
gsx_hip_status sorted_backward(const T* grad, int64_t grad_stride, const int32_t* ids, int64_t count, int64_t width,
                               float scale, float* out, int64_t table_rows, int64_t out_stride, int accumulate, void* temp,
                               hipStream_t stream) {
    const SortedIds at(count, table_rows, width);
    uint8_t* const base = static_cast<uint8_t*>(temp);
    KeyT* const keys = reinterpret_cast<KeyT*>(base + at.keys);
    KeyT* const sorted = reinterpret_cast<KeyT*>(base + at.keys_sorted);
    uint32_t* const order = reinterpret_cast<uint32_t*>(base + at.order);
    uint32_t* const starts = reinterpret_cast<uint32_t*>(base + at.starts);
    float* const partial = reinterpret_cast<float*>(base + at.partial);
    hipLaunchKernelGGL((lookup_keys_kernel<KeyT>), dim3(rows_grid(ceil_div(count, kRowThreads))), dim3(kRowThreads), 0,
                       stream, ids, count, (int32_t)table_rows, keys);
    int bits = 1;
    while ((table_rows >> bits) != 0) ++bits;
    const int passes = (bits + 7) / 8;
    const int digit = (bits + passes - 1) / passes;
    const gsx_hip_status st = tile_sort<KeyT>(keys, reinterpret_cast<KeyT*>(base + at.keys_alt), sorted,
                                              reinterpret_cast<uint32_t*>(base + at.order_alt), order, count, bits, passes,
                                              digit < 6 ? 6 : digit, base + at.sort, stream);
    if (st != GSX_HIP_SUCCESS) return fields_fail(st, "lookup backward: sort");
    hipLaunchKernelGGL((lookup_starts_kernel<KeyT>), dim3(rows_grid(ceil_div(table_rows + 1, kRowThreads))),
                       dim3(kRowThreads), 0, stream, sorted, count, table_rows, starts);
    const int64_t vecs = ceil_div(width, V);
    int lanes = 1;
    while (lanes < vecs && lanes < 64) lanes *= 2;
    // a wave takes 256 vectors of a row where the rows are that long, else its lanes share rows
    const int64_t groups = table_rows * ceil_div(vecs, vecs > 64 ? 256 : lanes);
    const int64_t parts = ceil_div(count, kRunPart) * ceil_div(vecs, lanes);
    const unsigned part_blocks = rows_grid(ceil_div(parts, kRowThreads / 64));
    const unsigned run_blocks = rows_grid(ceil_div(groups, kRowThreads / lanes));
    const auto runs = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(part_blocks + run_blocks), dim3(kRowThreads), 0, stream, grad, grad_stride, order,
                           sorted, starts, count, scale, out, table_rows, out_stride, width, lanes, accumulate, partial,
                           (int64_t)part_blocks);
    };
    if constexpr (V > 1) {
        if (vecs > 64) runs(lookup_runs_kernel<T, V, 4, KeyT>);
        else runs(lookup_runs_kernel<T, V, 1, KeyT>);
    } else {
        runs(lookup_runs_kernel<T, V, 1, KeyT>);  // rows of up to three columns
    }
    hipLaunchKernelGGL((lookup_join_kernel<V, KeyT>), dim3(rows_grid(parts)), dim3(kRowThreads), 0, stream, sorted, starts,
                       count, table_rows, width, lanes, partial, scale, out, out_stride, accumulate);
    return fields_launched("lookup backward launch");
}

}  // namespace

extern "C" {

gsx_hip_status gsx_hip_lookup_forward(const void* table, int32_t table_type, int64_t table_rows, int64_t table_stride,
                                      const int32_t* ids, int64_t count, int64_t width, float scale, void* out,
                                      int32_t out_type, int64_t out_stride, int* out_has_out_of_range,
                                      hipStream_t stream) {
    if (!known_type(table_type) || !known_type(out_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "lookup: rows are f32, bf16 or f16");
    if (!rows_fit(table_rows, table_stride, width) || !rows_fit(count, out_stride, width))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup: sizes must be >= 0 and strides >= width");
    if (count == 0 || width == 0) return GSX_HIP_SUCCESS;
    if (ids == nullptr || out == nullptr || (table == nullptr && table_rows > 0))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup: null pointer");
    if (!aligned_to(table, type_bytes(table_type)) || !aligned_to(out, type_bytes(out_type)) || !aligned_to(ids, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup: pointers must be aligned to their elements");
    return with_type(table_type, [&](auto t) {
        return with_type(out_type, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            constexpr int kMost = 16 / (int)(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
            const auto go = [&](auto launch) {
                return launch(table, table_rows, table_stride, ids, count, width, scale, out, out_stride,
                              out_has_out_of_range, stream);
            };
            // as many elements a thread as 16 bytes of the wider type hold, fewer in rows shorter than that
            if constexpr (kMost >= 8) {
                if (width >= 8) return go(launch_lookup<T, O, 8>);
            }
            if (width >= 4) return go(launch_lookup<T, O, 4>);
            if (width >= 2) return go(launch_lookup<T, O, 2>);
            return go(launch_lookup<T, O, 1>);
        });
    });
}

size_t gsx_hip_lookup_backward_temp_bytes(int64_t count, int64_t table_rows, int64_t width) {
    if (count <= 0 || table_rows <= 0 || width <= 0 || count > (int64_t)UINT32_MAX || table_rows > INT32_MAX ||
        takes_scan(count, table_rows, width))
        return 0;
    return (size_t)SortedIds(count, table_rows, width).bytes;
}

gsx_hip_status gsx_hip_lookup_backward(const void* grad_out, int32_t grad_type, int64_t grad_stride, const int32_t* ids,
                                       int64_t count, int64_t width, float scale, float* grad_table, int64_t table_rows,
                                       int64_t table_stride, int32_t accumulate, void* temp, hipStream_t stream) {
    if (!known_type(grad_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "lookup backward: rows are f32, bf16 or f16");
    if (!rows_fit(table_rows, table_stride, width) || !rows_fit(count, grad_stride, width))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup backward: sizes must be >= 0 and strides >= width");
    if (count > (int64_t)UINT32_MAX || table_rows > INT32_MAX)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "lookup backward: at most 2^32 - 1 ids and 2^31 - 1 table rows");
    if (table_rows == 0 || width == 0 || (count == 0 && accumulate != 0)) return GSX_HIP_SUCCESS;
    if (grad_table == nullptr || (count > 0 && (ids == nullptr || grad_out == nullptr)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup backward: null pointer");
    if (!aligned_to(grad_out, type_bytes(grad_type)) || !aligned_to(grad_table, 4) || !aligned_to(ids, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup backward: pointers must be aligned to their elements");
    const bool wide = width >= 4;  // columns a lane sums at once: four, or one of short rows
    if (takes_scan(count, table_rows, width)) {
        return with_type(grad_type, [&](auto t) {
            using T = decltype(t);
            const int64_t vecs = ceil_div(width, wide ? 4 : 1);
            const auto go = [&](auto kernel, int64_t blocks) {
                hipLaunchKernelGGL(kernel, dim3(rows_grid(blocks)), dim3(kRowThreads), 0, stream,
                                   static_cast<const T*>(grad_out), grad_stride, ids, count, scale, grad_table, table_rows,
                                   table_stride, width, accumulate);
            };
            const int64_t waves = table_rows * ceil_div(vecs, 64), long_waves = table_rows * ceil_div(vecs, 256);
            if (count > kScanSplit)
                go(wide ? lookup_scan_kernel<T, 4, 1, 4> : lookup_scan_kernel<T, 1, 1, 4>, waves);
            else if (vecs > 64 && long_waves >= kScanLong)
                go(lookup_scan_kernel<T, 4, 4, 1>, ceil_div(long_waves, 4));
            else
                go(wide ? lookup_scan_kernel<T, 4, 1, 1> : lookup_scan_kernel<T, 1, 1, 1>, ceil_div(waves, 4));
            return fields_launched("lookup backward launch");
        });
    }
    if (temp == nullptr || !aligned_to(temp, 16))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "lookup backward: the workspace must be non-null and 16-byte aligned");
    return with_type(grad_type, [&](auto t) {
        using T = decltype(t);
        const T* grad = static_cast<const T*>(grad_out);
        if (SortedIds::narrow(table_rows)) {
            return wide ? sorted_backward<T, 4, uint16_t>(grad, grad_stride, ids, count, width, scale, grad_table,
                                                                 table_rows, table_stride, accumulate, temp, stream)
                               : sorted_backward<T, 1, uint16_t>(grad, grad_stride, ids, count, width, scale, grad_table,
                                                                 table_rows, table_stride, accumulate, temp, stream);
        }
        return wide ? sorted_backward<T, 4, uint32_t>(grad, grad_stride, ids, count, width, scale, grad_table,
                                                             table_rows, table_stride, accumulate, temp, stream)
                           : sorted_backward<T, 1, uint32_t>(grad, grad_stride, ids, count, width, scale, grad_table,
                                                             table_rows, table_stride, accumulate, temp, stream);
    });
}

}  // extern "C"

// rows.hip - rows of a table looked up by id and scaled, and the table's gradient.
//
//   out[i, :] = s * table[id_i, :]            (an id outside the table: zeros)
//   G[v, :]   = s * sum over i with id_i = v of g[i, :]
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fields.hpp"

namespace gsx_amd {

constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;
constexpr int kRowTile = kRowThreads * kRowUnroll;  // vectors of V elements a workgroup copies at a time
constexpr int64_t kRowMostBlocks = 1 << 20;

// A tile is `tile_rows` whole rows of `vecs` vectors, or (vecs > kRowTile) a part of one row. Every id, then every row vector
// of a thread is loaded before the first store.
template <typename T, typename O, int V>
__global__ __launch_bounds__(kRowThreads) void lookup_kernel(const T* __restrict__ table, int64_t table_rows,
                                                             int64_t table_stride, const int32_t* __restrict__ ids,
                                                             int64_t count, int64_t vecs, int tile_rows, int64_t parts,
                                                             int64_t tiles, float scale, O* __restrict__ out,
                                                             int64_t out_stride, int* __restrict__ out_of_range) {
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row0 = tile / parts * tile_rows;
        const int64_t col0 = tile % parts * kRowTile;
        const uint32_t cols = (uint32_t)min(vecs - col0, (int64_t)kRowTile);
        const uint32_t work = (uint32_t)min((int64_t)tile_rows, count - row0) * cols;
        int32_t id[kRowUnroll];
        int64_t row[kRowUnroll], col[kRowUnroll];
        Vec<T, V> x[kRowUnroll];
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            const uint32_t e = threadIdx.x + u * kRowThreads;
            row[u] = row0 + e / cols;
            col[u] = (col0 + e % cols) * V;
            id[u] = e < work ? ids[row[u]] : -1;
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            if (id[u] >= 0 && id[u] < table_rows)
                x[u] = *reinterpret_cast<const Vec<T, V>*>(table + (int64_t)id[u] * table_stride + col[u]);
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; ++u) {
            if (threadIdx.x + u * kRowThreads >= work) continue;
            const bool fits = id[u] >= 0 && id[u] < table_rows;
            if (id[u] >= table_rows && out_of_range != nullptr) *out_of_range = 1;
            Vec<O, V> y;
#pragma unroll
            for (int k = 0; k < V; ++k) y.v[k] = from_float<O>(fits ? to_float(x[u].v[k]) * scale : 0.0f);
            *reinterpret_cast<Vec<O, V>*>(out + row[u] * out_stride + col[u]) = y;
        }
    }
}

// One wave per table row and 64 columns: it reads all ids, 64 at a time, and adds the rows of its id in ascending order.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void lookup_scan_kernel(const T* __restrict__ grad, int64_t grad_stride,
                                                                  const int32_t* __restrict__ ids, int64_t count,
                                                                  float scale, float* __restrict__ out,
                                                                  int64_t table_rows, int64_t out_stride, int64_t width,
                                                                  int accumulate) {
    const int lane = threadIdx.x & 63;
    const int64_t parts = (width + 63) / 64;
    const int64_t waves = table_rows * parts;
    for (int64_t w = (int64_t)blockIdx.x * (kRowThreads / 64) + threadIdx.x / 64; w < waves;
         w += (int64_t)gridDim.x * (kRowThreads / 64)) {
        const int64_t v = w / parts;
        const int64_t col = w % parts * 64 + lane;
        float sum = 0.0f;
        bool any = false;
        for (int64_t at = 0; at < count; at += 64) {
            const int32_t id = at + lane < count ? ids[at + lane] : -1;
            uint64_t mine = __builtin_amdgcn_ballot_w64(id == v);
            while (mine != 0) {
                const int k = __builtin_ctzll(mine);
                mine &= mine - 1;
                any = true;
                if (col < width) sum += to_float(grad[(at + k) * grad_stride + col]);
            }
        }
        if (col < width) {
            float* const p = out + v * out_stride + col;
            if (accumulate == 0) *p = sum * scale;
            else if (any) *p += sum * scale;
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

// Elements a thread moves at once: 16 bytes of the wider type where bases, strides and width allow it, else half of that, ...
int lookup_vector(const void* a, int32_t a_type, int64_t a_stride, const void* b, int32_t b_type, int64_t b_stride,
                  int64_t width) {
    const int64_t ab = type_bytes(a_type), bb = type_bytes(b_type);
    for (int64_t v = 16 / (ab > bb ? ab : bb); v > 1; v /= 2) {
        if (width % v == 0 && a_stride % v == 0 && b_stride % v == 0 && aligned_to(a, v * ab) && aligned_to(b, v * bb))
            return (int)v;
    }
    return 1;
}

template <typename T, typename O, int V>
gsx_hip_status launch_lookup(const void* table, int64_t table_rows, int64_t table_stride, const int32_t* ids,
                             int64_t count, int64_t width, float scale, void* out, int64_t out_stride, int* flag,
                             hipStream_t stream) {
    const int64_t vecs = width / V;
    const int tile_rows = vecs >= kRowTile ? 1 : (int)(kRowTile / vecs);
    const int64_t parts = ceil_div(vecs, kRowTile);
    const int64_t tiles = ceil_div(count, tile_rows) * parts;
    hipLaunchKernelGGL((lookup_kernel<T, O, V>), dim3((unsigned)(tiles < kRowMostBlocks ? tiles : kRowMostBlocks)),
                       dim3(kRowThreads), 0, stream, static_cast<const T*>(table), table_rows, table_stride, ids, count,
                       vecs, tile_rows, parts, tiles, scale, static_cast<O*>(out), out_stride, flag);
    return fields_launched("lookup launch");
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
    const int v = lookup_vector(table, table_type, table_stride, out, out_type, out_stride, width);
    return with_type(table_type, [&](auto t) {
        return with_type(out_type, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            constexpr int kMost = 16 / (int)(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
            const auto go = [&](auto launch) {
                return launch(table, table_rows, table_stride, ids, count, width, scale, out, out_stride,
                              out_has_out_of_range, stream);
            };
            if constexpr (kMost >= 8) {
                if (v == 8) return go(launch_lookup<T, O, 8>);
            }
            if (v == 4) return go(launch_lookup<T, O, 4>);
            if (v == 2) return go(launch_lookup<T, O, 2>);
            return go(launch_lookup<T, O, 1>);
        });
    });
}

size_t gsx_hip_lookup_backward_temp_bytes(int64_t count, int64_t table_rows, int64_t width) {
    (void)count;
    (void)table_rows;
    (void)width;
    return 0;
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
    (void)temp;
    return with_type(grad_type, [&](auto t) {
        using T = decltype(t);
        const int64_t blocks = ceil_div(table_rows * ceil_div(width, 64), kRowThreads / 64);
        hipLaunchKernelGGL((lookup_scan_kernel<T>), dim3((unsigned)(blocks < kRowMostBlocks ? blocks : kRowMostBlocks)),
                           dim3(kRowThreads), 0, stream, static_cast<const T*>(grad_out), grad_stride, ids, count, scale,
                           grad_table, table_rows, table_stride, width, accumulate);
        return fields_launched("lookup backward launch");
    });
}

}  // extern "C"

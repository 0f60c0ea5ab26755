// adamw.hip - AdamW over any number of tensors in one launch, its moments in float32 or in 8 bits.
//
// For every element, with t the steps so far and this one, in float32 (one rounding for each operation):
//   g = gradient * scale ;  m' = beta1 m + (1 - beta1) g ;  v' = beta2 v + (1 - beta2) (g g)
//   p' = p - (rate decay) p - (rate / (1 - beta1^t)) (m' / (sqrt(v') / sqrt(1 - beta2^t) + epsilon))
// The step count lives on the device: a launch of one workgroup counts it and forms each group's factors (in float64), so that
// the replays of a captured step count on.
//
// Moments in 8 bits are held in blocks of 128 elements of a tensor with a float32 scale for each block:
//   first:  s = max(max |m| * (1 / 448), 2^-126) ;  code = m * (1 / s) rounded to E4M3, ties to even
//   second: s = max(max v, 2^-126) ;  y = v * (1 / s) rounded to three bits behind the first, ties to even ;
//           code = (bits of y >> 20) - 762, at least 1 for v > 0 (1 stands for 1.375 * 2^-32, 254 for 1); 0 for v = 0
// Maxima are those of the finite values; what is not finite becomes NaN in the first moment, code 255 (+inf) in the second. The
// scales are not powers of two: as a block's largest value decays by less than half a step of its codes, the scale follows it.
// A second moment is never held as 0 unless it is: m' / sqrt(v') of a small value beside large ones stays bounded.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

#include "blocks.hpp"
#include "common.hpp"

namespace gsx_amd {

constexpr int kAdamwThreads = 256;
constexpr int kAdamwEach = 8;  // elements of a thread
constexpr int kAdamwChunk = kAdamwThreads * kAdamwEach;
constexpr int kHeld = 128;  // elements of a block of 8-bit moments: 16 threads
constexpr float kLeastScale = 0x1p-126f;
constexpr int kRatioBase = 762;  // code 254 is the ratio 1: its bits >> 20 are 1016

struct AdamwEntry {
    void* parameter;
    const void* gradient;
    void* first;
    void* second;
    float* first_scale;
    float* second_scale;
    int64_t count;
    int32_t parameter_type, gradient_type, bits, group;
};

// The table in device memory: this, the entries, then (entry, chunk of the entry) for each workgroup.
struct AdamwTable {
    int64_t entries, chunks;
    __host__ __device__ const AdamwEntry* entry_at(int64_t i) const { return reinterpret_cast<const AdamwEntry*>(this + 1) + i; }
};

struct AdamwRates {
    float beta1, new1, beta2, new2, decay, epsilon;
};
struct AdamwLaunch {
    AdamwRates rates[GSX_HIP_ADAM_MAX_GROUPS];
    float scale;
    const float* factor;  // may be null: 1
};
struct AdamwGroups {
    double beta1[GSX_HIP_ADAM_MAX_GROUPS], beta2[GSX_HIP_ADAM_MAX_GROUPS], rate[GSX_HIP_ADAM_MAX_GROUPS];
    int32_t count;
};
// What the step count decides, for each group: rate / (1 - beta1^t) and 1 / sqrt(1 - beta2^t).
struct AdamwFactors {
    float rate, root;
};

__global__ void adamw_count_kernel(AdamwGroups groups, int64_t* __restrict__ steps, AdamwFactors* __restrict__ factors) {
    const int64_t t = *steps + 1;
    __syncthreads();  // everybody has read it
    const int k = threadIdx.x;
    if (k < groups.count) {
        factors[k].rate = (float)(groups.rate[k] / (1.0 - pow(groups.beta1[k], (double)t)));
        factors[k].root = (float)(1.0 / sqrt(1.0 - pow(groups.beta2[k], (double)t)));
    }
    if (k == 0) *steps = t;
}

// Eight elements from `at` on as floats, zeros from `count` on.
template <typename T>
__device__ inline void load_eight(const T* __restrict__ p, int64_t at, int64_t count, float (&x)[8]) {
    const Raw<T, 8> r = load_raw<T, 8>(p, at, count);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = word_element<T>(r.w, i);
}
__device__ inline void load_eight(const void* p, int32_t type, int64_t at, int64_t count, float (&x)[8]) {
    if (type == GSX_HIP_DTYPE_F32) load_eight(static_cast<const float*>(p), at, count, x);
    else if (type == GSX_HIP_DTYPE_BF16) load_eight(static_cast<const __bf16*>(p), at, count, x);
    else load_eight(static_cast<const _Float16*>(p), at, count, x);
}

template <typename T>
__device__ inline void store_eight(T* __restrict__ p, int64_t at, int64_t count, const float (&x)[8]) {
    if (at + 8 <= count) {
        Octet<T> y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = from_float<T>(x[i]);
        *reinterpret_cast<Octet<T>*>(p + at) = y;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < count) p[at + i] = from_float<T>(x[i]);
    }
}
__device__ inline void store_eight(void* p, int32_t type, int64_t at, int64_t count, const float (&x)[8]) {
    if (type == GSX_HIP_DTYPE_F32) store_eight(static_cast<float*>(p), at, count, x);
    else if (type == GSX_HIP_DTYPE_BF16) store_eight(static_cast<__bf16*>(p), at, count, x);
    else store_eight(static_cast<_Float16*>(p), at, count, x);
}

typedef float v2f __attribute__((ext_vector_type(2)));

// First moments from their codes.
__device__ inline void first_four(uint32_t codes, float scale, float* m) {
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 1.0f, false);
    const v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 1.0f, true);
    m[0] = a[0] * scale;
    m[1] = a[1] * scale;
    m[2] = b[0] * scale;
    m[3] = b[1] * scale;
}
__device__ inline void first_values(uint2 codes, float scale, float (&m)[8]) {
    first_four(codes.x, scale, m);
    first_four(codes.y, scale, m + 4);
}

__device__ inline float second_value(uint32_t code, float scale) {
    const float y = __builtin_bit_cast(float, (code + kRatioBase) << 20);
    return code == 0 ? 0.0f : code == 255 ? INFINITY : y * scale;
}
__device__ inline void second_values(uint2 codes, float scale, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = second_value((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)) & 255u, scale);
}

// The largest of the 16 threads of a block.
__device__ inline float max_of_block(float v) {
    v = fmaxf(v, dpp_move<0xb1, 0xf>(v));
    v = fmaxf(v, dpp_move<0x4e, 0xf>(v));
    v = fmaxf(v, dpp_move<0x141, 0xf>(v));
    return fmaxf(v, dpp_move<0x140, 0xf>(v));
}

// Codes of a block's values, eight a thread, and its scale.
__device__ inline uint2 hold_first(const float (&m)[8], float& scale) {
    float top = 0.0f;
    bool special = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool finite = finite_bits(__builtin_bit_cast(uint32_t, m[i]));
        special |= !finite;
        top = fmaxf(top, finite ? fabsf(m[i]) : 0.0f);
    }
    top = max_of_block(top);
    scale = fmaxf(top * (1.0f / 448.0f), kLeastScale);
    const float inverse = 1.0f / scale;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_fmed3f(m[i] * inverse, -448.0f, 448.0f);
    uint2 codes = make_uint2(pack_finite(x, 1.0f), pack_finite(x + 4, 1.0f));
    if (special) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t bits = __builtin_bit_cast(uint32_t, m[i]);
            if (finite_bits(bits)) continue;
            uint32_t& word = i < 4 ? codes.x : codes.y;  // NaN with the sign of what is there
            word = (word & ~(0xffu << (8 * (i & 3)))) | (0x7fu | (bits >> 31 << 7)) << (8 * (i & 3));
        }
    }
    return codes;
}

__device__ inline uint2 hold_second(const float (&v)[8], float& scale) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_bits(__builtin_bit_cast(uint32_t, v[i])) ? v[i] : 0.0f);
    top = max_of_block(top);
    scale = fmaxf(top, kLeastScale);
    const float inverse = 1.0f / scale;
    uint2 codes = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, v[i] * inverse);
        int code = (int)((bits + 0x7ffffu + (bits >> 20 & 1u)) >> 20) - kRatioBase;
        code = min(max(code, 1), 254);
        if (v[i] <= 0.0f) code = 0;
        if (!finite_bits(__builtin_bit_cast(uint32_t, v[i]))) code = 255;
        (i < 4 ? codes.x : codes.y) |= (uint32_t)code << (8 * (i & 3));
    }
    return codes;
}

// A workgroup takes 2048 elements of one tensor, found in the table, so that tensors of any sizes fill the GPU in one launch; a thread
// eight of them, whose moments in 8 bits are one load each, and 16 threads a block, whose largest value four lane exchanges find.
// Bound by memory: 105M elements in 48 tensors, gradients of 16 bits and moments of 8, 267 to 279 us one step after another (5.3 to
// 5.6 TB/s; the vector units are never idle either), 256 between calls that read the moments; 4.7M in 61 tensors of 16 bits 21 us
// (4.9 TB/s), 576000 in two tensors 6 us, its latency.
__global__ __launch_bounds__(kAdamwThreads) void adamw_kernel(const AdamwTable* __restrict__ table, AdamwLaunch launch,
                                                              int32_t group_count,
                                                              const AdamwFactors* __restrict__ factors) {
    if ((int64_t)blockIdx.x >= table->chunks) return;
    const uint2 chunk = reinterpret_cast<const uint2*>(table->entry_at(table->entries))[blockIdx.x];
    const AdamwEntry e = *table->entry_at(chunk.x);
    if (e.group >= group_count) return;
    const AdamwRates r = launch.rates[e.group];
    const AdamwFactors f = factors[e.group];
    const float scale = launch.scale * (launch.factor != nullptr ? *launch.factor : 1.0f);
    const int64_t at = (int64_t)chunk.y * kAdamwChunk + threadIdx.x * kAdamwEach;
    float p[8], g[8], m[8], v[8];
    load_eight(e.parameter, e.parameter_type, at, e.count, p);
    load_eight(e.gradient, e.gradient_type, at, e.count, g);
    const bool held = e.bits == 8;
    if (held) {
        // whole blocks are there whatever the count is; behind it they are 0
        uint2 first = make_uint2(0u, 0u), second = first;
        float first_scale = 0.0f, second_scale = 0.0f;
        if (at < e.count) {
            first = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(e.first) + at);
            second = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(e.second) + at);
            first_scale = e.first_scale[at / kHeld];
            second_scale = e.second_scale[at / kHeld];
        }
        first_values(first, first_scale, m);
        second_values(second, second_scale, v);
    } else {
        load_eight(static_cast<const float*>(e.first), at, e.count, m);
        load_eight(static_cast<const float*>(e.second), at, e.count, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = g[i] * scale;
        m[i] = r.beta1 * m[i] + r.new1 * x;
        v[i] = r.beta2 * v[i] + r.new2 * (x * x);
        const float change = m[i] / (sqrtf(v[i]) * f.root + r.epsilon);
        p[i] = p[i] - r.decay * p[i] - f.rate * change;
    }
    store_eight(e.parameter, e.parameter_type, at, e.count, p);
    if (held) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (at + i < e.count) continue;
            m[i] = 0.0f;
            v[i] = 0.0f;
        }
        float first_scale, second_scale;
        const uint2 first = hold_first(m, first_scale), second = hold_second(v, second_scale);
        if (at < (e.count + kHeld - 1) / kHeld * kHeld) {
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(e.first) + at) = first;
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(e.second) + at) = second;
            if (at % kHeld == 0) {
                e.first_scale[at / kHeld] = first_scale;
                e.second_scale[at / kHeld] = second_scale;
            }
        }
    } else {
        store_eight(static_cast<float*>(e.first), at, e.count, m);
        store_eight(static_cast<float*>(e.second), at, e.count, v);
    }
}

// Whole blocks of moments from float32, 16 threads a block, and back: 16 bytes a thread and store, which pass the caches by. Bound by
// memory. 105M pairs of moments: held 182 us, 5.6 TB/s; read 145, 7.1 TB/s, call after call (259 with 32 bytes a thread in two stores
// through the caches), and 208 to 213, 4.9 TB/s, right behind a step, where programs read them.
constexpr int kReadEach = 4;  // fours of a thread
constexpr int kReadFours = kAdamwThreads * kReadEach;

__global__ __launch_bounds__(kAdamwThreads) void moments_hold_kernel(const float* __restrict__ first,
                                                                     const float* __restrict__ second, int64_t blocks,
                                                                     uint8_t* __restrict__ first_codes,
                                                                     float* __restrict__ first_scale,
                                                                     uint8_t* __restrict__ second_codes,
                                                                     float* __restrict__ second_scale) {
    for (int64_t b = (int64_t)blockIdx.x * (kAdamwThreads / 16) + threadIdx.x / 16; b < blocks;
         b += (int64_t)gridDim.x * (kAdamwThreads / 16)) {
        const int64_t at = b * kHeld + (threadIdx.x & 15) * 8;
        float x[8], s;
        load_eight(first, at, blocks * kHeld, x);
        *reinterpret_cast<uint2*>(first_codes + at) = hold_first(x, s);
        if ((threadIdx.x & 15) == 0) first_scale[b] = s;
        load_eight(second, at, blocks * kHeld, x);
        *reinterpret_cast<uint2*>(second_codes + at) = hold_second(x, s);
        if ((threadIdx.x & 15) == 0) second_scale[b] = s;
    }
}

__global__ __launch_bounds__(kAdamwThreads) void moments_read_kernel(const uint8_t* __restrict__ first_codes,
                                                                     const float* __restrict__ first_scale,
                                                                     const uint8_t* __restrict__ second_codes,
                                                                     const float* __restrict__ second_scale, int64_t blocks,
                                                                     float* __restrict__ first, float* __restrict__ second) {
    typedef float v4f __attribute__((ext_vector_type(4)));
    struct __attribute__((packed, aligned(4))) Loose {
        v4f v;
    };
    const auto store = [](float* to, const float (&x)[4]) {
        __builtin_nontemporal_store(v4f{x[0], x[1], x[2], x[3]}, &reinterpret_cast<Loose*>(to)->v);
    };
    const int64_t fours = blocks * (kHeld / 4);
    for (int64_t b = blockIdx.x; b * kReadFours < fours; b += gridDim.x) {
        uint32_t m[kReadEach], v[kReadEach];
        float s[kReadEach], t[kReadEach];
#pragma unroll
        for (int u = 0; u < kReadEach; ++u) {
            const int64_t i = min(b * kReadFours + u * kAdamwThreads + threadIdx.x, fours - 1);
            m[u] = reinterpret_cast<const uint32_t*>(first_codes)[i];
            v[u] = reinterpret_cast<const uint32_t*>(second_codes)[i];
            s[u] = first_scale[i / (kHeld / 4)];
            t[u] = second_scale[i / (kHeld / 4)];
        }
#pragma unroll
        for (int u = 0; u < kReadEach; ++u) {
            const int64_t i = b * kReadFours + u * kAdamwThreads + threadIdx.x;
            if (i >= fours) break;
            float x[4];
            first_four(m[u], s[u], x);
            store(first + 4 * i, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = second_value(v[u] >> (8 * j) & 255u, t[u]);
            store(second + 4 * i, x);
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

constexpr int64_t kAdamwMostChunks = (1 << 24) - 1;  // a launch has less than 2^32 threads

// Chunks of all tensors; -1: a tensor is not one that a step takes (the message says why).
int64_t adamw_chunks(const gsx_hip_adamw_tensor* tensors, int64_t count) {
    const auto refuse = [](gsx_hip_status code, const char* what) {
        fields_fail(code, what);
        return (int64_t)code;
    };
    if (count < 0 || count > INT32_MAX || (count > 0 && tensors == nullptr))
        return refuse(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: 0 to 2^31 - 1 tensors");
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        const gsx_hip_adamw_tensor& t = tensors[i];
        if (!known_type(t.parameter_type) || !known_type(t.gradient_type))
            return refuse(GSX_HIP_ERROR_NOT_SUPPORTED, "adamw: parameters and gradients are f32, bf16 or f16");
        if (t.bits != 8 && t.bits != 32) return refuse(GSX_HIP_ERROR_NOT_SUPPORTED, "adamw: moments have 8 bits or 32");
        if (t.count < 0 || t.group < 0 || t.group >= GSX_HIP_ADAM_MAX_GROUPS)
            return refuse(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: counts must be >= 0 and groups 0 to 15");
        if (t.count == 0) continue;
        if (t.count > kAdamwMostChunks * kAdamwChunk)
            return refuse(GSX_HIP_ERROR_OUT_OF_RANGE, "adamw: a step takes at most 2^24 - 1 chunks of 2048 elements");
        if (t.parameter == nullptr || t.gradient == nullptr || t.first == nullptr || t.second == nullptr ||
            (t.bits == 8 && (t.first_scale == nullptr || t.second_scale == nullptr)))
            return refuse(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: null pointer");
        if (!aligned_to(t.parameter, type_bytes(t.parameter_type)) || !aligned_to(t.gradient, type_bytes(t.gradient_type)) ||
            !aligned_to(t.first, t.bits == 8 ? 8 : 4) || !aligned_to(t.second, t.bits == 8 ? 8 : 4) ||
            (t.bits == 8 && (!aligned_to(t.first_scale, 4) || !aligned_to(t.second_scale, 4))))
            return refuse(GSX_HIP_ERROR_INVALID_ARGUMENT,
                          "adamw: pointers must be aligned to their elements, 8-bit moments to 8 bytes");
        chunks += ceil_div(t.count, kAdamwChunk);
        if (chunks > kAdamwMostChunks)
            return refuse(GSX_HIP_ERROR_OUT_OF_RANGE, "adamw: a step takes at most 2^24 - 1 chunks of 2048 elements");
    }
    return chunks;
}

// Whether nothing that a step writes is read or written under another name.
bool adamw_apart(const gsx_hip_adamw_tensor* tensors, int64_t count) {
    struct Span {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Span> spans;
    spans.reserve((size_t)count * 6);
    const auto add = [&](const void* p, int64_t bytes, bool written) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(p);
        spans.push_back({from, from + (uintptr_t)bytes, written});
    };
    for (int64_t i = 0; i < count; ++i) {
        const gsx_hip_adamw_tensor& t = tensors[i];
        if (t.count == 0) continue;
        const int64_t blocks = ceil_div(t.count, kHeld), moments = t.bits == 8 ? blocks * kHeld : t.count * 4;
        add(t.parameter, t.count * type_bytes(t.parameter_type), true);
        add(t.gradient, t.count * type_bytes(t.gradient_type), false);
        add(t.first, moments, true);
        add(t.second, moments, true);
        if (t.bits == 8) {
            add(t.first_scale, blocks * 4, true);
            add(t.second_scale, blocks * 4, true);
        }
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    uintptr_t end = 0, written_end = 0;  // of the spans before
    for (const Span& s : spans) {
        if (s.from < (s.written ? end : written_end)) return false;
        end = std::max(end, s.to);
        if (s.written) written_end = std::max(written_end, s.to);
    }
    return true;
}

}  // namespace

extern "C" {

size_t gsx_hip_adamw_table_bytes(const gsx_hip_adamw_tensor* tensors, int64_t tensor_count) {
    const int64_t chunks = adamw_chunks(tensors, tensor_count);
    if (chunks < 0) return 0;
    return sizeof(AdamwTable) + (size_t)tensor_count * sizeof(AdamwEntry) + (size_t)chunks * 8;
}

gsx_hip_status gsx_hip_adamw_table_fill(const gsx_hip_adamw_tensor* tensors, int64_t tensor_count, void* table,
                                        int64_t* out_chunks) {
    const int64_t chunks = adamw_chunks(tensors, tensor_count);
    if (chunks < 0) return (gsx_hip_status)chunks;
    if (table == nullptr || out_chunks == nullptr || !aligned_to(table, 8))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: the table must be non-null and 8-byte aligned");
    try {
        if (!adamw_apart(tensors, tensor_count))
            return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: what a step writes may not overlap anything else of it");
    } catch (...) {
        return fields_fail(GSX_HIP_ERROR_OUT_OF_MEMORY, "adamw: no host memory");
    }
    AdamwTable* const head = static_cast<AdamwTable*>(table);
    head->entries = tensor_count;
    head->chunks = chunks;
    AdamwEntry* const entries = const_cast<AdamwEntry*>(head->entry_at(0));
    uint32_t* chunk = reinterpret_cast<uint32_t*>(entries + tensor_count);
    for (int64_t i = 0; i < tensor_count; ++i) {
        const gsx_hip_adamw_tensor& t = tensors[i];
        entries[i] = {t.parameter, t.gradient, t.first, t.second, t.first_scale, t.second_scale, t.count,
                      t.parameter_type, t.gradient_type, t.bits, t.group};
        for (int64_t c = 0; c < ceil_div(t.count, kAdamwChunk); ++c) {
            *chunk++ = (uint32_t)i;
            *chunk++ = (uint32_t)c;
        }
    }
    *out_chunks = chunks;
    return GSX_HIP_SUCCESS;
}

gsx_hip_status gsx_hip_adamw_step(const void* table, int64_t chunks, const gsx_hip_adamw_group* groups, int32_t group_count,
                                  float grad_scale, const float* grad_factor, int64_t* steps, void* factors,
                                  hipStream_t stream) {
    if (groups == nullptr || group_count < 1 || group_count > GSX_HIP_ADAM_MAX_GROUPS)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "adamw: 1 to 16 groups");
    if (chunks < 0 || chunks > kAdamwMostChunks)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "adamw: a step takes at most 2^24 - 1 chunks of 2048 elements");
    if (table == nullptr || steps == nullptr || factors == nullptr || !aligned_to(table, 8) || !aligned_to(steps, 8) ||
        !aligned_to(factors, 8) || !aligned_to(grad_factor, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "adamw: table, step count and factors must be non-null and 8-byte aligned");
    AdamwLaunch launch = {};
    AdamwGroups counted = {};
    launch.scale = grad_scale;
    launch.factor = grad_factor;
    counted.count = group_count;
    for (int k = 0; k < group_count; ++k) {
        const gsx_hip_adamw_group& g = groups[k];
        if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0) || !((float)g.epsilon > 0.0f) ||
            !(g.weight_decay >= 0.0) || !std::isfinite(g.learning_rate) || !std::isfinite(g.weight_decay))
            return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                               "adamw: 0 <= beta < 1, epsilon > 0, weight decay >= 0, a finite learning rate");
        launch.rates[k] = {(float)g.beta1, (float)(1.0 - g.beta1), (float)g.beta2, (float)(1.0 - g.beta2),
                           (float)(g.learning_rate * g.weight_decay), (float)g.epsilon};
        counted.beta1[k] = g.beta1;
        counted.beta2[k] = g.beta2;
        counted.rate[k] = g.learning_rate;
    }
    AdamwFactors* const f = static_cast<AdamwFactors*>(factors);
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(64), 0, stream, counted, steps, f);
    if (chunks > 0)
        hipLaunchKernelGGL(adamw_kernel, dim3((unsigned)chunks), dim3(kAdamwThreads), 0, stream,
                           static_cast<const AdamwTable*>(table), launch, group_count, f);
    return fields_launched("adamw launch");
}

static gsx_hip_status moments_check(const void* first_codes, const float* first_scale, const void* second_codes,
                                    const float* second_scale, int64_t blocks, const float* first, const float* second) {
    if (blocks < 0 || blocks > INT64_MAX / (8 * kHeld))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "moments: the number of blocks must be >= 0");
    if (blocks > 0 && (first_codes == nullptr || first_scale == nullptr || second_codes == nullptr ||
                       second_scale == nullptr || first == nullptr || second == nullptr))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "moments: null pointer");
    if (!aligned_to(first_codes, 8) || !aligned_to(second_codes, 8) || !aligned_to(first_scale, 4) ||
        !aligned_to(second_scale, 4) || !aligned_to(first, 4) || !aligned_to(second, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "moments: codes must be 8-byte aligned, floats 4-byte");
    return GSX_HIP_SUCCESS;
}

gsx_hip_status gsx_hip_moments_hold(const float* first, const float* second, int64_t blocks, uint8_t* first_codes,
                                    float* first_scale, uint8_t* second_codes, float* second_scale, hipStream_t stream) {
    const gsx_hip_status st = moments_check(first_codes, first_scale, second_codes, second_scale, blocks, first, second);
    if (st != GSX_HIP_SUCCESS || blocks == 0) return st;
    hipLaunchKernelGGL(moments_hold_kernel, dim3(blocks_grid(ceil_div(blocks, kAdamwThreads / 16))), dim3(kAdamwThreads), 0,
                       stream, first, second, blocks, first_codes, first_scale, second_codes, second_scale);
    return fields_launched("moments launch");
}

gsx_hip_status gsx_hip_moments_read(const uint8_t* first_codes, const float* first_scale, const uint8_t* second_codes,
                                    const float* second_scale, int64_t blocks, float* first, float* second,
                                    hipStream_t stream) {
    const gsx_hip_status st = moments_check(first_codes, first_scale, second_codes, second_scale, blocks, first, second);
    if (st != GSX_HIP_SUCCESS || blocks == 0) return st;
    hipLaunchKernelGGL(moments_read_kernel, dim3(blocks_grid(ceil_div(blocks * (kHeld / 4), kReadFours))), dim3(kAdamwThreads), 0,
                       stream, first_codes, first_scale, second_codes, second_scale, blocks, first, second);
    return fields_launched("moments launch");
}

}  // extern "C"

// distill.hip - distillation from a teacher's top logits: loss and gradient.
//
// One row: z [vocab] the student's logits, (id_k, t_k) the teacher's top entries, T the temperature, w the row's weight.
//   p = softmax(t / T) over the valid entries (id in the vocabulary, t not -inf),  q = softmax(z / T) over the whole row
//   loss = w T^2 sum_k p_k (log p_k - log q_{id_k})
//   dz_j = c w T (q_j - sum_{k: id_k = j} p_k)
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.hpp"
#include "fields.hpp"

namespace gsx_amd {

// Maximum m of a set of logits and sum s of exp((z - m) / T), joined over disjoint sets. m = -inf: nothing above -inf (s = 0). A
// NaN or +inf among the logits leaves a NaN in s: (z - m) / T is one.
struct MaxSum {
    float m, s;
};

constexpr int kDistillMostTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    int64_t rows, vocab, logits_stride, grad_stride, teacher_stride;
    const int32_t* ids;
    const float* teacher;
    int32_t top;
    float temperature;
    float scale2;             // log2(e) / temperature
    const float* row_weight;  // may be null: 1
    const float* row_grad;    // may be null: 1
    float grad_scale;
    float* loss;              // may be null
    float* stats;             // may be null where it is written
    int32_t from_stats;       // read them instead of forming them
    int64_t first_row;        // of a launch over a part of the rows
    int64_t slice, slices;    // logits of a workgroup where a row has several, and how many
    MaxSum* partial;
};

__device__ inline float exp2_scaled(float x, float m, float scale2) { return __builtin_amdgcn_exp2f((x - m) * scale2); }

__device__ inline MaxSum join(MaxSum a, MaxSum b, float scale2) {
    MaxSum r;
    r.m = fmaxf(a.m, b.m);
    const float base = r.m == -INFINITY ? 0.0f : r.m;
    r.s = a.s * exp2_scaled(a.m, base, scale2) + b.s * exp2_scaled(b.m, base, scale2);
    return r;
}

// A group of kGroup threads works on one row: 16 lanes of a wave, a wave of its own, or the whole workgroup.
template <int kGroup>
__device__ inline void group_sync() {
    if constexpr (kGroup <= 64) wave_lds_sync();
    else __syncthreads();
}

// Sum and maximum over a group; s_wave holds a float for each of the group's waves. NaN does not pass max_of_group (fmaxf).
__device__ inline float wave_reduce_max(float v) {  // lane moves as in wave_reduce_sum; NaN is passed over
    v = fmaxf(v, dpp_move<0xb1, 0xf>(v));
    v = fmaxf(v, dpp_move<0x4e, 0xf>(v));
    v = fmaxf(v, dpp_move<0x141, 0xf>(v));
    v = fmaxf(v, dpp_move<0x140, 0xf>(v));
    v = fmaxf(v, dpp_move<0x142, 0xa>(v));  // lanes that get nothing here do not reach lane 63
    v = fmaxf(v, dpp_move<0x143, 0xc>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <int kGroup>
__device__ inline float sum_of_group(float v, float* s_wave) {
    if constexpr (kGroup == 16) {
        v += dpp_move<0xb1, 0xf>(v);
        v += dpp_move<0x4e, 0xf>(v);
        v += dpp_move<0x141, 0xf>(v);
        return v + dpp_move<0x140, 0xf>(v);
    }
    v = wave_reduce_sum(v);
    if constexpr (kGroup == 64) return v;
    const int wave = threadIdx.x / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[wave] = v;
    __syncthreads();
    v = s_wave[0];
#pragma unroll
    for (int w = 1; w < kGroup / 64; ++w) v += s_wave[w];
    return v;
}

template <int kGroup>
__device__ inline float max_of_group(float v, float* s_wave) {
    if constexpr (kGroup == 16) {
        v = fmaxf(v, dpp_move<0xb1, 0xf>(v));
        v = fmaxf(v, dpp_move<0x4e, 0xf>(v));
        v = fmaxf(v, dpp_move<0x141, 0xf>(v));
        return fmaxf(v, dpp_move<0x140, 0xf>(v));
    }
    v = wave_reduce_max(v);
    if constexpr (kGroup == 64) return v;
    const int wave = threadIdx.x / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[wave] = v;
    __syncthreads();
    v = s_wave[0];
#pragma unroll
    for (int w = 1; w < kGroup / 64; ++w) v = fmaxf(v, s_wave[w]);
    return v;
}

// The teacher's side of one row: in LDS for each entry its id (-1: does not count), its logit, its p and the student's logit
// there.
struct Teacher {
    int32_t* id;
    float* t;
    float* p;
    float* z;
    uint16_t* slot;      // of a row of a wave or less: an entry that names each logit
    bool unique;         // no id is known to be named twice
    float max, log_sum;  // log p_k = (t_k - max) / T - log_sum
    bool any;            // an entry counts
};

// Loads what teacher_finish needs; between the two the caller may load its part of the row.
template <typename T, int kGroup>
__device__ inline void teacher_load(const DistillArgs& a, const T* __restrict__ z, int64_t row, int tid, Teacher& r) {
    const int32_t* ids = a.ids + row * a.teacher_stride;
    const float* t = a.teacher + row * a.teacher_stride;
    for (int k = tid; k < a.top; k += kGroup) {
        const int32_t id = ids[k];
        const float x = t[k];
        const bool counts = id >= 0 && id < a.vocab && !(x == -INFINITY);
        r.id[k] = counts ? id : -1;
        r.t[k] = x;
        r.z[k] = counts ? to_float(z[id]) : 0.0f;
    }
}

template <int kGroup>
__device__ inline void teacher_finish(const DistillArgs& a, int tid, float* s_wave, Teacher& r, bool want_unique) {
    float m = -INFINITY, any = 0.0f;
    for (int k = tid; k < a.top; k += kGroup) {
        if (r.id[k] < 0) continue;
        m = fmaxf(m, r.t[k]);
        any = 1.0f;
    }
    m = max_of_group<kGroup>(m, s_wave);
    const float inv_t = 1.0f / a.temperature;
    float sum = 0.0f;
    for (int k = tid; k < a.top; k += kGroup) {
        const float e = r.id[k] >= 0 ? expf((r.t[k] - m) * inv_t) : 0.0f;  // NaN stays NaN, in the sum too
        r.p[k] = e;
        sum += e;
    }
    r.any = max_of_group<kGroup>(any, s_wave) != 0.0f;
    sum = sum_of_group<kGroup>(sum, s_wave);
    r.max = m;
    r.log_sum = logf(sum);
    for (int k = tid; k < a.top; k += kGroup) r.p[k] = r.any ? r.p[k] / sum : 0.0f;
    r.unique = false;
    if constexpr (kGroup <= 64) {  // whoever wrote a slot last finds itself there; an id named twice leaves somebody else
        if (want_unique) {
            for (int k = tid; k < a.top; k += kGroup)
                if (r.id[k] >= 0) r.slot[r.id[k]] = (uint16_t)k;
            group_sync<kGroup>();
            bool twice = false;
            for (int k = tid; k < a.top; k += kGroup) twice |= r.id[k] >= 0 && r.slot[r.id[k]] != (uint16_t)k;
            if constexpr (kGroup == 64) r.unique = wave_none(twice);
            else r.unique = (__builtin_amdgcn_ballot_w64(twice) >> (threadIdx.x & 48) & 0xffffu) == 0;
        }
    }
    group_sync<kGroup>();
}

// sum_k p_k (log p_k - log q_{id_k}) by the group (every thread returns it).
template <int kGroup>
__device__ inline float cross_terms(const DistillArgs& a, int tid, const Teacher& r, float* s_wave, MaxSum q) {
    const float inv_t = 1.0f / a.temperature;
    const float log_s = logf(q.s);
    float sum = 0.0f;
    for (int k = tid; k < a.top; k += kGroup) {
        if (r.id[k] < 0 || r.p[k] == 0.0f) continue;
        const float log_p = (r.t[k] - r.max) * inv_t - r.log_sum;
        const float x = r.z[k];
        const float log_q = x == -INFINITY && !(q.s != q.s) ? -INFINITY : (x - q.m) * inv_t - log_s;
        sum += r.p[k] * (log_p - log_q);
    }
    return sum_of_group<kGroup>(sum, s_wave);
}

// The gradient of logit z with softmax numerator and denominator from q: base = q.m, cq = c / q.s.
__device__ inline float q_term(float z, float base, float cq, float scale2) { return cq * exp2_scaled(z, base, scale2); }

// The teacher's entries with ids in [from, to) again, with all their p: after the group's stores of c q_j. c = 0 and a row
// without a distribution need none.
template <typename T, int kGroup>
__device__ inline void patch_entries(const DistillArgs& a, T* __restrict__ g, int64_t from, int64_t to, int tid,
                                     const Teacher& r, float base, float cq, float c) {
    for (int k = tid; k < a.top; k += kGroup) {
        const int32_t id = r.id[k];
        if (id < from || id >= to || id < 0) continue;
        float p = r.p[k];
        if (!r.unique) {  // an id that is named twice has both
            p = 0.0f;
            for (int o = 0; o < a.top; ++o) p += r.id[o] == id ? r.p[o] : 0.0f;
        }
        g[id] = from_float<T>(q_term(r.z[k], base, cq, a.scale2) - c * p);
    }
}

// 16 bytes of logits at any element's address.
template <typename T>
struct Words {
    static constexpr int kElements = 16 / (int)sizeof(T);
    uint32_t w[4];
};
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) LooseWords {
    uint32_t w[4];
};

template <typename T>
__device__ inline float element_of(const Words<T>& x, int i) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(float, x.w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
        return __builtin_bit_cast(float, i & 1 ? x.w[i / 2] & 0xffff0000u : x.w[i / 2] << 16);
    } else {
        return to_float(__builtin_bit_cast(T, (uint16_t)(i & 1 ? x.w[i / 2] >> 16 : x.w[i / 2])));
    }
}

// Keeps the compiler from holding what it unpacked or computed from x beside x itself until the next use: registers are what
// bounds the rows that fit.
template <typename T>
__device__ inline void repack(Words<T>& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(x.w[i]));
}

template <typename T>
__device__ inline uint32_t element_bits(float x) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, x);
    else return __builtin_bit_cast(uint16_t, from_float<T>(x));
}

// Vector v of a row, -inf in all its elements where there is none (v >= vecs).
template <typename T>
__device__ inline Words<T> load_words(const T* __restrict__ z, int v, int vecs) {
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __bf16) ? 0xff80ff80u : 0xfc00fc00u;
    Words<T> x = {{kNone, kNone, kNone, kNone}};
    if (v < vecs) {
        const LooseWords<T> y = *reinterpret_cast<const LooseWords<T>*>(z + (uint32_t)v * Words<T>::kElements);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.w[i] = y.w[i];
    }
    return x;
}

template <typename T>
__device__ inline void store_words(T* __restrict__ g, int v, int vecs, const float (&y)[Words<T>::kElements]) {
    if (v >= vecs) return;
    LooseWords<T> x;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.w[i] = element_bits<T>(y[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.w[i] = element_bits<T>(y[2 * i]) | element_bits<T>(y[2 * i + 1]) << 16;
    }
    typedef uint32_t Loose2 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t Loose4 __attribute__((ext_vector_type(4), aligned(4)));
    const Loose4 y4 = {x.w[0], x.w[1], x.w[2], x.w[3]};
    if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(y4, reinterpret_cast<Loose4*>(g + (uint32_t)v * Words<T>::kElements));
    else __builtin_nontemporal_store(y4, reinterpret_cast<Loose2*>(g + (uint32_t)v * Words<T>::kElements));
}

// A stretch of `length` logits at z: `lead` elements up to the first address that is a multiple of 16, then `vecs` vectors, then
// fewer than a vector. What is before and behind the vectors is taken one a thread (fewer than 16 threads): `loose` is a
// thread's element or -1. Vectors that are not aligned cost a fifth (rows of 65537 bf16: 271 against 237 us).
struct Stretch {
    int lead, vecs;
    int64_t loose;
};

template <typename T>
__device__ inline Stretch stretch_of(const T* z, int64_t length, int tid) {
    constexpr int kElements = Words<T>::kElements;
    Stretch s;
    s.lead = (int)min((int64_t)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int64_t)sizeof(T), length);
    s.vecs = (int)((length - s.lead) / kElements);
    const int64_t behind = s.lead + (int64_t)s.vecs * kElements + (tid - s.lead);
    s.loose = tid < s.lead ? tid : behind < length ? behind : -1;
    return s;
}

// Rows that fit the registers of a group: kGroup threads hold kVecs times 16 bytes each. The logits are read once; maximum, sum
// and gradient come from registers. Instructions bound short rows (307200 of 150 bf16: 81 us, 2.5 TB/s, vector instructions in
// 98% of the cycles), memory bounds long ones (4096 of 65537 bf16: 1.07 GB in 234 us, 4.6 TB/s, a copy's rate). The loss alone
// takes 52 and 113 us, the gradient in a later call 65 and 235 more.
template <typename T, int kGroup, int kVecs>
__global__ __launch_bounds__(kGroup < 256 ? 256 : kGroup) void distill_held_kernel(DistillArgs a, const T* __restrict__ logits,
                                                                                   T* __restrict__ grad) {
    constexpr int kGroups = kGroup < 256 ? 256 / kGroup : 1;  // rows of a workgroup
    constexpr int kElements = Words<T>::kElements;
    extern __shared__ uint8_t s_distill[];
    __shared__ float s_wave[16];
    const int group = kGroups == 1 ? 0 : threadIdx.x / kGroup, tid = kGroups == 1 ? threadIdx.x : threadIdx.x % kGroup;
    Teacher r;
    r.id = reinterpret_cast<int32_t*>(s_distill) + group * 4 * a.top;
    r.t = reinterpret_cast<float*>(r.id + a.top);
    r.p = r.t + a.top;
    r.z = r.p + a.top;
    r.slot = reinterpret_cast<uint16_t*>(s_distill + kGroups * 16 * a.top) + group * a.vocab;
    for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < a.rows; row += (int64_t)gridDim.x * kGroups) {
        const T* const z = logits + row * a.logits_stride;
        const float w = a.row_weight != nullptr ? a.row_weight[row] : 1.0f;
        const Stretch st = stretch_of<T>(z, a.vocab, tid);
        Words<T> x[kVecs];
        group_sync<kGroup>();  // the row before has been patched
#pragma unroll
        for (int u = 0; u < kVecs; ++u) x[u] = load_words<T>(z + st.lead + u * kGroup * kElements, tid, st.vecs - u * kGroup);
        const float last = st.loose >= 0 ? to_float(z[st.loose]) : -INFINITY;
        teacher_load<T, kGroup>(a, z, row, tid, r);
        MaxSum q;
        if (a.from_stats != 0) {
            q.m = a.stats[2 * row];
            q.s = a.stats[2 * row + 1];
        } else {
            float m = last == last ? last : -INFINITY;
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
#pragma unroll
                for (int i = 0; i < kElements; ++i) m = fmaxf(m, element_of(x[u], i));
            q.m = max_of_group<kGroup>(m, s_wave);
            const float base = q.m == -INFINITY ? 0.0f : q.m;
            float s = exp2_scaled(last, base, a.scale2);
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                repack(x[u]);
#pragma unroll
                for (int i = 0; i < kElements; ++i) s += exp2_scaled(element_of(x[u], i), base, a.scale2);
            }
            q.s = sum_of_group<kGroup>(s, s_wave);
        }
        teacher_finish<kGroup>(a, tid, s_wave, r, grad != nullptr);
        const bool live = r.any && w != 0.0f;
        if (a.from_stats == 0) {
            const float terms = cross_terms<kGroup>(a, tid, r, s_wave, q);
            if (tid == 0) {
                if (a.loss != nullptr) a.loss[row] = live ? w * a.temperature * a.temperature * terms : 0.0f;
                if (a.stats != nullptr) {
                    a.stats[2 * row] = q.m;
                    a.stats[2 * row + 1] = q.s;
                }
            }
        }
        if (grad == nullptr) continue;
        T* const g = grad + row * a.grad_stride;
        const bool some = live && q.s != 0.0f;
        const float c = (a.row_grad != nullptr ? a.row_grad[row] : 1.0f) * a.grad_scale * w * a.temperature;
        const float cq = some ? c / q.s : 0.0f, base = q.m == -INFINITY ? 0.0f : q.m;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            float y[kElements];
            repack(x[u]);
#pragma unroll
            for (int i = 0; i < kElements; ++i)
                y[i] = some ? q_term(element_of(x[u], i), base, cq, a.scale2) : 0.0f;
            store_words<T>(g + st.lead + u * kGroup * kElements, tid, st.vecs - u * kGroup, y);
        }
        if (st.loose >= 0) g[st.loose] = from_float<T>(some ? q_term(last, base, cq, a.scale2) : 0.0f);
        if (some) {
            group_sync<kGroup>();  // orders those stores before the entries'
            patch_entries<T, kGroup>(a, g, 0, a.vocab, tid, r, base, cq, c);
        }
    }
}

// Longer rows, and few of them: a row is cut into slices of a workgroup each. This launch leaves every slice's maximum and sum,
constexpr int kSliceThreads = 256;

template <typename T>
__global__ __launch_bounds__(kSliceThreads) void distill_slices_kernel(DistillArgs a, const T* __restrict__ logits) {
    __shared__ float s_wave[kSliceThreads / 64];
    constexpr int kElements = Words<T>::kElements, kAhead = 4;
    const int64_t total = a.rows * a.slices;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t row = a.first_row + b / a.slices, from = b % a.slices * a.slice;
        const int64_t to = min(from + a.slice, a.vocab);
        const T* const z = logits + row * a.logits_stride + from;
        const Stretch st = stretch_of<T>(z, to - from, threadIdx.x);
        MaxSum q = {-INFINITY, 0.0f};
        if (st.loose >= 0) {
            const float last = to_float(z[st.loose]);
            q.m = last == last ? last : -INFINITY;
            q.s = exp2_scaled(last, q.m == -INFINITY ? 0.0f : q.m, a.scale2);
        }
        for (int v = threadIdx.x; v < st.vecs; v += kSliceThreads * kAhead) {
            Words<T> x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) x[u] = load_words<T>(z + st.lead, v + u * kSliceThreads, st.vecs);
            float m = q.m;
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int i = 0; i < kElements; ++i) m = fmaxf(m, element_of(x[u], i));
            const float base = m == -INFINITY ? 0.0f : m;
            float s = q.s * exp2_scaled(q.m, base, a.scale2);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int i = 0; i < kElements; ++i) s += exp2_scaled(element_of(x[u], i), base, a.scale2);
            q = {m, s};
        }
        const float m = max_of_group<kSliceThreads>(q.m, s_wave);
        const float base = m == -INFINITY ? 0.0f : m;
        const float s = sum_of_group<kSliceThreads>(q.s * exp2_scaled(q.m, base, a.scale2), s_wave);
        if (threadIdx.x == 0) a.partial[b] = {m, s};
    }
}

// and this one joins them (every workgroup of a row does), writes the loss (the first slice's) and the gradient. One row of 131072
// float32: 3 and 9 us, chains of barriers and loads rather than bytes.
template <typename T>
__global__ __launch_bounds__(kSliceThreads) void distill_finish_kernel(DistillArgs a, const T* __restrict__ logits,
                                                                       T* __restrict__ grad, int64_t slices_run) {
    extern __shared__ uint8_t s_distill[];
    __shared__ float s_wave[kSliceThreads / 64];
    constexpr int kElements = Words<T>::kElements, kAhead = 4;
    Teacher r;
    r.id = reinterpret_cast<int32_t*>(s_distill);
    r.t = reinterpret_cast<float*>(r.id + a.top);
    r.p = r.t + a.top;
    r.z = r.p + a.top;
    r.slot = nullptr;
    const int64_t total = a.rows * slices_run;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t local = b / slices_run, row = a.first_row + local, from = b % slices_run * a.slice;
        const int64_t to = min(from + a.slice, a.vocab);
        const T* const z = logits + row * a.logits_stride;
        const float w = a.row_weight != nullptr ? a.row_weight[row] : 1.0f;
        __syncthreads();  // the slice before has been patched
        teacher_load<T, kSliceThreads>(a, z, row, threadIdx.x, r);
        // the slice's first vectors are on their way while the sums are joined
        const Stretch st = stretch_of<T>(z + from, to - from, threadIdx.x);
        Words<T> x[kAhead];
        float last = -INFINITY;
        if (grad != nullptr) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                x[u] = load_words<T>(z + from + st.lead, threadIdx.x + u * kSliceThreads, st.vecs);
            if (st.loose >= 0) last = to_float(z[from + st.loose]);
        }
        MaxSum q = {-INFINITY, 0.0f};
        if (a.from_stats != 0) {
            q.m = a.stats[2 * row];
            q.s = a.stats[2 * row + 1];
        } else {
            for (int64_t i = threadIdx.x; i < a.slices; i += kSliceThreads) q = join(q, a.partial[local * a.slices + i], a.scale2);
            const float m = max_of_group<kSliceThreads>(q.m, s_wave);
            const float base = m == -INFINITY ? 0.0f : m;
            q.s = sum_of_group<kSliceThreads>(q.s * exp2_scaled(q.m, base, a.scale2), s_wave);
            q.m = m;
        }
        teacher_finish<kSliceThreads>(a, threadIdx.x, s_wave, r, false);
        const bool live = r.any && w != 0.0f;
        if (a.from_stats == 0 && from == 0) {
            const float terms = cross_terms<kSliceThreads>(a, threadIdx.x, r, s_wave, q);
            if (threadIdx.x == 0) {
                if (a.loss != nullptr) a.loss[row] = live ? w * a.temperature * a.temperature * terms : 0.0f;
                if (a.stats != nullptr) {
                    a.stats[2 * row] = q.m;
                    a.stats[2 * row + 1] = q.s;
                }
            }
        }
        if (grad == nullptr) continue;
        T* const g = grad + row * a.grad_stride;
        const bool some = live && q.s != 0.0f;
        const float c = (a.row_grad != nullptr ? a.row_grad[row] : 1.0f) * a.grad_scale * w * a.temperature;
        const float cq = some ? c / q.s : 0.0f, base = q.m == -INFINITY ? 0.0f : q.m;
        for (int v = threadIdx.x; v < st.vecs; v += kSliceThreads * kAhead) {
            if (v != (int)threadIdx.x) {
#pragma unroll
                for (int u = 0; u < kAhead; ++u) x[u] = load_words<T>(z + from + st.lead, v + u * kSliceThreads, st.vecs);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float y[kElements];
#pragma unroll
                for (int i = 0; i < kElements; ++i) y[i] = some ? q_term(element_of(x[u], i), base, cq, a.scale2) : 0.0f;
                store_words<T>(g + from + st.lead, v + u * kSliceThreads, st.vecs, y);
            }
        }
        if (st.loose >= 0) g[from + st.loose] = from_float<T>(some ? q_term(last, base, cq, a.scale2) : 0.0f);
        if (some) {
            __syncthreads();  // orders those stores before the entries'
            patch_entries<T, kSliceThreads>(a, g, from, to, threadIdx.x, r, base, cq, c);
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

gsx_hip_status distill_check(const DistillArgs& a, const void* logits, int32_t type, const void* grad) {
    if (!known_type(type)) return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "distill: logits are f32, bf16 or f16");
    if (a.vocab < 1 || a.vocab > INT32_MAX || a.top < 1 || a.top > kDistillMostTop)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "distill: 1 to 2^31 - 1 logits a row and 1 to 1024 teacher entries");
    if (!rows_fit(a.rows, a.logits_stride, a.vocab) || !rows_fit(a.rows, a.teacher_stride, a.top) ||
        (grad != nullptr && !rows_fit(a.rows, a.grad_stride, a.vocab)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: rows must be >= 0 and strides at least the row's length");
    if (!(a.temperature >= 1e-6f) || !(a.temperature <= 1e6f))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: the temperature must lie between 1e-6 and 1e6");
    if (a.rows > 0 && (logits == nullptr || a.ids == nullptr || a.teacher == nullptr))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: null pointer");
    if (!aligned_to(logits, type_bytes(type)) || !aligned_to(grad, type_bytes(type)) || !aligned_to(a.ids, 4) ||
        !aligned_to(a.teacher, 4) || !aligned_to(a.row_weight, 4) || !aligned_to(a.row_grad, 4) ||
        !aligned_to(a.loss, 4) || !aligned_to(a.stats, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: pointers must be aligned to their elements");
    if (logits != nullptr && logits == grad)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: the gradient may not overwrite the logits");
    return GSX_HIP_SUCCESS;
}

// A row is held by 16 lanes of a wave (up to 1 KB, and 1792 bytes of LDS), by a wave (4 KB), by 256 threads (64 KB), 512 (128 KB)
// or 1024 (256 KB): the smallest group that holds it in 16 vectors a thread, so that two or more rows share a CU and one loads
// while another is computed. 307200 rows of 150 bf16 with 8 entries: a wave took 2.6 times as long as 16 lanes; 100000 of 512
// with 64 entries, 2 KB of LDS: 16 lanes 97 us, a wave 91. 4096 rows of 65536 bf16: 512 threads 227 us, 1024 with half the
// vectors each 289. Above 32 KB only where there are rows enough for the GPU's 256 CUs; else, and beyond, a row is cut into
// slices of 16 KB or more, so that some 2048 workgroups share the logits.
struct DistillPlan {
    int group, vecs;        // group = 0: slices
    int64_t slice, slices;  // logits of a slice
    int64_t batch;          // rows of a pair of launches: what they read twice stays in the 256 MB cache between
};

DistillPlan distill_plan(int64_t rows, int64_t vocab, int64_t bytes, int64_t top) {
    DistillPlan p = {};
    const int64_t vecs = vocab * bytes / 16;  // the few elements behind the last whole vector are held besides
    if (vecs <= 16 * 4 && 16 * top + 2 * vocab <= 1792) p.group = 16;
    else if (vecs <= 64 * 4) p.group = 64;
    else if (vecs <= 256 * 8 || (vecs <= 256 * 16 && rows >= 192)) p.group = 256;
    else if (vecs <= 512 * 16 && rows >= 192) p.group = 512;
    else if (vecs <= 1024 * 16 && rows >= 192) p.group = 1024;
    if (p.group != 0) {
        p.vecs = vecs > 0 ? (int)ceil_div(vecs, p.group) : 1;
        p.batch = rows;
        return p;
    }
    const int64_t least = 16384 / bytes;
    p.batch = ceil_div((int64_t)128 << 20, vocab * bytes);
    if (p.batch > rows) p.batch = rows;
    int64_t slices = ceil_div(2048, p.batch);
    if (slices > vocab / least) slices = vocab / least;
    if (slices < 1) slices = 1;
    p.slice = ceil_div(ceil_div(vocab, slices), 2048) * 2048;
    p.slices = ceil_div(vocab, p.slice);
    return p;
}

template <typename T, int kGroup, int kVecs>
gsx_hip_status launch_held(const DistillArgs& a, const T* logits, T* grad, hipStream_t stream) {
    const int per = kGroup < 256 ? 256 / kGroup : 1;
    const int64_t blocks = ceil_div(a.rows, per);
    hipLaunchKernelGGL((distill_held_kernel<T, kGroup, kVecs>), dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)),
                       dim3(kGroup < 256 ? 256 : kGroup), (unsigned)(per * (16 * a.top + (kGroup <= 64 ? 2 * a.vocab : 0))),
                       stream, a, logits, grad);
    return fields_launched("distill launch");
}

template <typename T>
gsx_hip_status launch_distill(const DistillPlan& p, DistillArgs a, const T* logits, T* grad, void* temp,
                              hipStream_t stream) {
    if (p.group == 16) {
        if (p.vecs <= 1) return launch_held<T, 16, 1>(a, logits, grad, stream);
        if (p.vecs <= 2) return launch_held<T, 16, 2>(a, logits, grad, stream);
        return launch_held<T, 16, 4>(a, logits, grad, stream);
    }
    if (p.group == 64) {
        if (p.vecs <= 1) return launch_held<T, 64, 1>(a, logits, grad, stream);
        if (p.vecs <= 2) return launch_held<T, 64, 2>(a, logits, grad, stream);
        return launch_held<T, 64, 4>(a, logits, grad, stream);
    }
    if (p.group == 256) {
        if (p.vecs <= 2) return launch_held<T, 256, 2>(a, logits, grad, stream);
        if (p.vecs <= 4) return launch_held<T, 256, 4>(a, logits, grad, stream);
        if (p.vecs <= 8) return launch_held<T, 256, 8>(a, logits, grad, stream);
        if (p.vecs <= 12) return launch_held<T, 256, 12>(a, logits, grad, stream);
        return launch_held<T, 256, 16>(a, logits, grad, stream);
    }
    if (p.group == 512) {
        if (p.vecs <= 12) return launch_held<T, 512, 12>(a, logits, grad, stream);
        return launch_held<T, 512, 16>(a, logits, grad, stream);
    }
    if (p.group == 1024) {
        if (p.vecs <= 12) return launch_held<T, 1024, 12>(a, logits, grad, stream);
        return launch_held<T, 1024, 16>(a, logits, grad, stream);
    }
    const int64_t rows = a.rows;
    a.slice = p.slice;
    a.slices = p.slices;
    a.partial = static_cast<MaxSum*>(temp);
    const int64_t run = grad != nullptr ? p.slices : 1;
    const auto grid = [](int64_t blocks) { return dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)); };
    for (a.first_row = 0; a.first_row < rows; a.first_row += p.batch) {
        a.rows = rows - a.first_row < p.batch ? rows - a.first_row : p.batch;
        if (a.from_stats == 0)
            hipLaunchKernelGGL((distill_slices_kernel<T>), grid(a.rows * p.slices), dim3(kSliceThreads), 0, stream, a, logits);
        hipLaunchKernelGGL((distill_finish_kernel<T>), grid(a.rows * run), dim3(kSliceThreads), (unsigned)(16 * a.top), stream,
                           a, logits, grad, run);
    }
    return fields_launched("distill launch");
}

gsx_hip_status distill_launch(const DistillPlan& p, const DistillArgs& a, const void* logits, int32_t type, void* grad,
                              void* temp, hipStream_t stream) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return launch_distill<T>(p, a, static_cast<const T*>(logits), static_cast<T*>(grad), temp, stream);
    });
}

DistillArgs distill_args(int64_t logits_stride, int64_t rows, int64_t vocab, const int32_t* ids, const float* teacher,
                         int64_t teacher_stride, int32_t top, float temperature, const float* row_weight) {
    DistillArgs a = {};
    a.rows = rows;
    a.vocab = vocab;
    a.logits_stride = logits_stride;
    a.teacher_stride = teacher_stride;
    a.ids = ids;
    a.teacher = teacher;
    a.top = top;
    a.temperature = temperature;
    a.scale2 = kLog2e / temperature;
    a.row_weight = row_weight;
    return a;
}

}  // namespace

extern "C" {

size_t gsx_hip_distill_temp_bytes(int64_t rows, int64_t vocab) {
    if (rows <= 0 || vocab <= 0 || vocab > INT32_MAX) return 0;
    int64_t most = 0;  // whatever the logits' type is
    for (int64_t bytes = 2; bytes <= 4; bytes += 2) {
        const DistillPlan p = distill_plan(rows, vocab, bytes, 1);
        const int64_t need = p.group != 0 ? 0 : p.batch * p.slices * (int64_t)sizeof(MaxSum);
        if (need > most) most = need;
    }
    return (size_t)most;
}

gsx_hip_status gsx_hip_distill_forward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                       int64_t vocab, const int32_t* teacher_ids, const float* teacher_logits,
                                       int64_t teacher_stride, int32_t top, float temperature, const float* row_weight,
                                       float* loss, float* row_stats, void* grad_logits, int64_t grad_stride,
                                       float grad_scale, void* temp, hipStream_t stream) {
    DistillArgs a = distill_args(logits_stride, rows, vocab, teacher_ids, teacher_logits, teacher_stride, top, temperature,
                                 row_weight);
    a.grad_stride = grad_stride;
    a.grad_scale = grad_scale;
    a.loss = loss;
    a.stats = row_stats;
    const gsx_hip_status st = distill_check(a, logits, logits_type, grad_logits);
    if (st != GSX_HIP_SUCCESS || rows == 0) return st;
    const DistillPlan p = distill_plan(rows, vocab, type_bytes(logits_type), top);
    if (p.group == 0 && (temp == nullptr || !aligned_to(temp, 16)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill: the workspace must be non-null and 16-byte aligned");
    return distill_launch(p, a, logits, logits_type, grad_logits, temp, stream);
}

gsx_hip_status gsx_hip_distill_backward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                        int64_t vocab, const int32_t* teacher_ids, const float* teacher_logits,
                                        int64_t teacher_stride, int32_t top, float temperature, const float* row_weight,
                                        const float* row_stats, const float* row_grad, float grad_scale,
                                        void* grad_logits, int64_t grad_stride, hipStream_t stream) {
    DistillArgs a = distill_args(logits_stride, rows, vocab, teacher_ids, teacher_logits, teacher_stride, top, temperature,
                                 row_weight);
    a.grad_stride = grad_stride;
    a.grad_scale = grad_scale;
    a.row_grad = row_grad;
    a.stats = const_cast<float*>(row_stats);  // read only
    const gsx_hip_status st = distill_check(a, logits, logits_type, grad_logits);
    if (st != GSX_HIP_SUCCESS || rows == 0) return st;
    if (row_stats == nullptr || grad_logits == nullptr)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "distill backward: null pointer");
    a.from_stats = 1;
    return distill_launch(distill_plan(rows, vocab, type_bytes(logits_type), top), a, logits, logits_type, grad_logits, nullptr,
                          stream);
}

}  // extern "C"

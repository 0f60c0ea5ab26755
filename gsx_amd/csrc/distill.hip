// distill.hip - distillation from a teacher's top logits: loss and gradient.
//
// One row: z [vocab] the student's logits, (id_k, t_k) the teacher's top entries, T the temperature, w the row's weight.
//   p = softmax(t / T) over the valid entries (id in the vocabulary, t not -inf),  q = softmax(z / T) over the whole row
//   loss = w T^2 sum_k p_k (log p_k - log q_{id_k})
//   dz_j = c w T (q_j - sum_{k: id_k = j} p_k)
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fields.hpp"

namespace gsx_amd {

constexpr int kDistillThreads = 256;
constexpr int kDistillMostTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    int64_t rows, vocab, logits_stride, grad_stride, teacher_stride;
    const int32_t* ids;
    const float* teacher;
    int32_t top;
    float temperature;
    float scale2;            // log2(e) / temperature
    const float* row_weight; // may be null: 1
    const float* row_grad;   // may be null: 1
    float grad_scale;
    float* loss;
    float* stats;
};

// Maximum m of a set of logits and sum s of exp((z - m) / T), joined over disjoint sets. m = -inf: nothing yet (s = 0). A NaN
// or +inf among the logits leaves a NaN in s.
struct MaxSum {
    float m, s;
};

__device__ inline float exp2_scaled(float x, float m, float scale2) { return __builtin_amdgcn_exp2f((x - m) * scale2); }

__device__ inline MaxSum join(MaxSum a, MaxSum b, float scale2) {
    MaxSum r;
    r.m = fmaxf(a.m, b.m);
    const float base = r.m == -INFINITY ? 0.0f : r.m;
    r.s = a.s * exp2_scaled(a.m, base, scale2) + b.s * exp2_scaled(b.m, base, scale2);
    return r;
}

__device__ inline MaxSum wave_join(MaxSum a, float scale2) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        MaxSum b;
        b.m = __shfl_xor(a.m, off, 64);
        b.s = __shfl_xor(a.s, off, 64);
        a = join(a, b, scale2);
    }
    return a;
}

// The teacher's side of one row in LDS, by the whole workgroup: s_id (-1: not valid) and s_p (p_k); true if there is a valid
// entry. log p_k = (t_k - m) / T - log_sum. Ends with a barrier.
template <int kThreads>
__device__ inline bool teacher_row(const DistillArgs& a, int64_t row, int32_t* s_id, float* s_p, float* s_wave,
                                   float& t_max, float& log_sum) {
    const int32_t* ids = a.ids + row * a.teacher_stride;
    const float* t = a.teacher + row * a.teacher_stride;
    float m = -INFINITY;
    bool nan = false;
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const int32_t id = ids[k];
        const float x = t[k];
        const bool valid = id >= 0 && id < a.vocab && !(x == -INFINITY);
        s_id[k] = valid ? id : -1;
        s_p[k] = x;
        if (valid) {
            m = fmaxf(m, x);
            nan |= x != x;
        }
    }
    if (nan) m = NAN;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float o = __shfl_xor(m, off, 64);
        m = m != m || o != o ? NAN : fmaxf(m, o);
    }
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x / 64] = m;
    __syncthreads();
    m = s_wave[0];
    for (int w = 1; w < kThreads / 64; ++w) m = m != m || s_wave[w] != s_wave[w] ? NAN : fmaxf(m, s_wave[w]);
    t_max = m;
    const bool any = !(m == -INFINITY);
    const float inv_t = 1.0f / a.temperature;
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const float e = s_id[k] >= 0 ? expf((s_p[k] - m) * inv_t) : 0.0f;
        s_p[k] = e;
        sum += e;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    __syncthreads();  // s_wave has been read
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x / 64] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < kThreads / 64; ++w) sum += s_wave[w];
    log_sum = logf(sum);
    for (int k = threadIdx.x; k < a.top; k += kThreads) s_p[k] = any ? s_p[k] / sum : 0.0f;
    __syncthreads();
    return any;
}

// sum_k p_k (log p_k - log q_{id_k}) of one row by the whole workgroup (every thread returns it).
template <typename T, int kThreads>
__device__ inline float cross_terms(const DistillArgs& a, const T* z, int64_t row, const int32_t* s_id, const float* s_p,
                                    float* s_wave, float t_max, float log_sum, MaxSum q) {
    const float* t = a.teacher + row * a.teacher_stride;
    const float inv_t = 1.0f / a.temperature;
    const float log_s = logf(q.s);
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        if (s_id[k] < 0 || s_p[k] == 0.0f) continue;
        const float log_p = (t[k] - t_max) * inv_t - log_sum;
        const float x = to_float(z[s_id[k]]);
        const float log_q = x == -INFINITY && !(q.s != q.s) ? -INFINITY : (x - q.m) * inv_t - log_s;
        sum += s_p[k] * (log_p - log_q);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x / 64] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < kThreads / 64; ++w) sum += s_wave[w];
    return sum;
}

// Gradient of a row by the whole workgroup: every logit's q_j first, then the teacher's entries again with all their p_k.
template <typename T, int kThreads>
__device__ inline void write_grad(const DistillArgs& a, const T* z, T* g, const int32_t* s_id, const float* s_p, MaxSum q,
                                  bool live, float c) {
    const float base = q.m == -INFINITY ? 0.0f : q.m;
    if (!live || q.s == 0.0f) {
        for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) g[j] = from_float<T>(0.0f);
        return;
    }
    const float cq = c / q.s;
    for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads)
        g[j] = from_float<T>(cq * exp2_scaled(to_float(z[j]), base, a.scale2));
    __syncthreads();  // orders these stores before the entries' below
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const int32_t id = s_id[k];
        if (id < 0) continue;
        float p = 0.0f;
        for (int o = 0; o < a.top; ++o) p += s_id[o] == id ? s_p[o] : 0.0f;
        g[id] = from_float<T>(cq * exp2_scaled(to_float(z[id]), base, a.scale2) - c * p);
    }
}

// One workgroup per row: maximum and sum in one pass over the logits, then (grad) a second pass.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_row_kernel(DistillArgs a, const T* __restrict__ logits,
                                                                      T* __restrict__ grad, int from_stats) {
    __shared__ int32_t s_id[kDistillMostTop];
    __shared__ float s_p[kDistillMostTop];
    __shared__ float s_wave[2 * kDistillThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = logits + row * a.logits_stride;
        float t_max, log_sum;
        const bool any = teacher_row<kDistillThreads>(a, row, s_id, s_p, s_wave, t_max, log_sum);
        const float w = a.row_weight != nullptr ? a.row_weight[row] : 1.0f;
        const bool live = any && w != 0.0f;
        MaxSum q = {-INFINITY, 0.0f};
        if (from_stats != 0) {
            q.m = a.stats[2 * row];
            q.s = a.stats[2 * row + 1];
        } else {
            for (int64_t j = threadIdx.x; j < a.vocab; j += kDistillThreads) {
                MaxSum one = {to_float(z[j]), 1.0f};
                if (one.m == -INFINITY) one.s = 0.0f;
                if (one.m != one.m) one = {-INFINITY, NAN};
                q = join(q, one, a.scale2);
            }
            q = wave_join(q, a.scale2);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                s_wave[2 * (threadIdx.x / 64)] = q.m;
                s_wave[2 * (threadIdx.x / 64) + 1] = q.s;
            }
            __syncthreads();
            q = {s_wave[0], s_wave[1]};
            for (int i = 1; i < kDistillThreads / 64; ++i) q = join(q, {s_wave[2 * i], s_wave[2 * i + 1]}, a.scale2);
            __syncthreads();
            const float terms = cross_terms<T, kDistillThreads>(a, z, row, s_id, s_p, s_wave, t_max, log_sum, q);
            if (threadIdx.x == 0) {
                if (a.loss != nullptr) a.loss[row] = live ? w * a.temperature * a.temperature * terms : 0.0f;
                if (a.stats != nullptr) {
                    a.stats[2 * row] = q.m;
                    a.stats[2 * row + 1] = q.s;
                }
            }
        }
        if (grad != nullptr) {
            const float c = (a.row_grad != nullptr ? a.row_grad[row] : 1.0f) * a.grad_scale * w * a.temperature;
            write_grad<T, kDistillThreads>(a, z, grad + row * a.grad_stride, s_id, s_p, q, live, c);
        }
        __syncthreads();
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

gsx_hip_status distill_launch(const DistillArgs& a, const void* logits, int32_t type, void* grad, int from_stats,
                              hipStream_t stream) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((distill_row_kernel<T>), dim3((unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20))),
                           dim3(kDistillThreads), 0, stream, a, static_cast<const T*>(logits), static_cast<T*>(grad),
                           from_stats);
        return fields_launched("distill launch");
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
    (void)rows;
    (void)vocab;
    return 0;
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
    (void)temp;
    return distill_launch(a, logits, logits_type, grad_logits, 0, stream);
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
    return distill_launch(a, logits, logits_type, grad_logits, 1, stream);
}

}  // extern "C"

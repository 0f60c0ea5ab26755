// logits.hpp - rows of logits in registers, for distill.hip and logprobs.hip: vectors of them at any element's address, sums and
// maxima over the threads that share a row.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.hpp"
#include "fields.hpp"

namespace gsx_amd {

constexpr float kLog2e = 1.4426950408889634f;

// Maximum m of a set of logits and sum s of exp((z - m) / T), joined over disjoint sets. m = -inf: nothing above -inf (s = 0). A
// NaN or +inf among the logits leaves a NaN in s: (z - m) / T is one.
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

// A vector of logits, 16 bytes unless said otherwise, at any element's address.
template <typename T, int kWords = 4>
struct Words {
    static constexpr int kElements = 4 * kWords / (int)sizeof(T);
    uint32_t w[kWords];
};
template <typename T, int kWords>
struct __attribute__((packed, aligned(sizeof(T)))) LooseWords {
    uint32_t w[kWords];
};

template <typename T, int kWords>
__device__ inline float element_of(const Words<T, kWords>& x, int i) {
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
template <typename T, int kWords>
__device__ inline void repack(Words<T, kWords>& x) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(x.w[i]));
}

template <typename T>
__device__ inline uint32_t element_bits(float x) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, x);
    else return __builtin_bit_cast(uint16_t, from_float<T>(x));
}

// Vector v of a row, -inf in all its elements where there is none (v >= vecs).
template <typename T, int kWords = 4>
__device__ inline Words<T, kWords> load_words(const T* __restrict__ z, int v, int vecs) {
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __bf16) ? 0xff80ff80u : 0xfc00fc00u;
    Words<T, kWords> x;
#pragma unroll
    for (int i = 0; i < kWords; ++i) x.w[i] = kNone;
    if (v < vecs) {
        const LooseWords<T, kWords> y =
            *reinterpret_cast<const LooseWords<T, kWords>*>(z + (uint32_t)v * Words<T, kWords>::kElements);
#pragma unroll
        for (int i = 0; i < kWords; ++i) x.w[i] = y.w[i];
    }
    return x;
}

// Past the caches, unless a line is written by several stores (kPast false; 8 lanes of 8 bytes, 307200 x 150: 45 us, past them 72).
template <typename T, int kWords = 4, bool kPast = true>
__device__ inline void store_words(T* __restrict__ g, int v, int vecs, const float (&y)[Words<T, kWords>::kElements]) {
    if (v >= vecs) return;
    LooseWords<T, kWords> x;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x.w[i] = element_bits<T>(y[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x.w[i] = element_bits<T>(y[2 * i]) | element_bits<T>(y[2 * i + 1]) << 16;
    }
    typedef uint32_t Loose2 __attribute__((ext_vector_type(kWords), aligned(2)));
    typedef uint32_t Loose4 __attribute__((ext_vector_type(kWords), aligned(4)));
    const Loose4 all = __builtin_bit_cast(Loose4, x);
    T* const to = g + (uint32_t)v * Words<T, kWords>::kElements;
    if constexpr (!kPast) *reinterpret_cast<Loose2*>(to) = all;
    else if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(all, reinterpret_cast<Loose4*>(to));
    else __builtin_nontemporal_store(all, reinterpret_cast<Loose2*>(to));
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

}  // namespace gsx_amd

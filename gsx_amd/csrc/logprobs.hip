// logprobs.hip - log probabilities of given labels, entropies and top alternatives of rows of logits, and their gradient.
//
// One row: z [vocab], T the temperature, y = z / T, q = softmax(y), id the given label:
//   chosen = log q_id,  entropy H = -sum_j q_j log q_j,  top: the largest z (of equal ones the lowest index) with their log q
//   dz_j = (gl (delta_{j,id} - q_j) - gh q_j (log q_j + H)) / T   for upstream gradients gl of chosen and gh of H
// With m = max z, u_j = (z_j - m) log2(e) / T and e_j = 2^u_j, all of it follows from s = sum e_j and w = sum e_j u_j:
//   log q_j = ln2 u_j - ln s,  H = ln s - ln2 w / s    (terms of one sign: nothing cancels)
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "logits.hpp"

namespace gsx_amd {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMostAlternatives = 64;
constexpr float kLeastExponent2 = -256.0f;  // 2 to this is 0, a float's least is 2^-149

// Of a set of logits: m, s and w as above.
struct RowSums {
    float m, s, w;
};

struct LogProbsArgs {
    int64_t rows, vocab, logits_stride, grad_stride;
    const int32_t* ids;  // may be null
    float inv_t;
    float scale2;  // log2(e) / temperature
    float* chosen;   // may be null
    float* entropy;  // may be null
    float* stats;    // may be null: m, s, H
    bool backward;   // stats are read, only the gradient is written
    int32_t top;
    int32_t* top_ids;
    float* top_logs;
    const float* row_grad;      // may be null: 1
    const float* entropy_grad;  // may be null: 1
    float grad_scale, entropy_scale;
    int64_t slice, slices;  // logits of a workgroup where a row has several, and how many
    RowSums* partial;       // of each slice
    uint64_t* partial_top;  // [slice][top] keys
};

// u_j where e_j is not 0, and finite for z_j = -inf, so that e_j u_j = 0 there. NaN is left to e_j.
__device__ inline float scaled_from(float z, float base, float scale2) { return fmaxf((z - base) * scale2, kLeastExponent2); }

// Whole numbers in the order of the logits: NaN above everything, -0 with 0. 0 is below all of them, 2^32 - 1 above.
__device__ inline uint32_t ordered_number(float x) {  // of a number, or NaN without a sign
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ inline uint32_t ordered_bits(float x) { return x != x ? 0xfffffffeu : ordered_number(x); }
__device__ inline float ordered_value(uint32_t o) {
    return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
constexpr uint32_t kOrderedClosed = 0x007fffffu;  // of -inf

// The order of the alternatives: by value, then by the lowest index; 0: none. Rows of few logits in 16-bit types have 32 bits for it.
__device__ inline uint64_t key_of(float x, int64_t index) {
    return (uint64_t)ordered_bits(x) << 32 | (0xffffffffu - (uint32_t)index);
}
__device__ inline bool key_open(uint64_t key) { return (uint32_t)(key >> 32) > kOrderedClosed; }

template <typename T>
struct RowKey {
    typedef uint64_t Type;
    static __device__ inline Type of(float x, int index) { return key_of(x, index); }
    static __device__ inline Type of_number(float x, int index) {
        return (uint64_t)ordered_number(x) << 32 | (0xffffffffu - (uint32_t)index);
    }
    static __device__ inline uint64_t wide(Type k) { return key_open(k) ? k : 0; }
};
// A float32 that holds a 16-bit one has zeros in its last 13 bits: the index (of at most 2^13 logits) takes their place.
struct ShortRowKey {
    typedef uint32_t Type;
    static __device__ inline Type with(uint32_t order, int index) { return (order & ~0x1fffu) | (0x1fffu - (uint32_t)index); }
    static __device__ inline Type of(float x, int index) { return with(ordered_bits(x), index); }
    static __device__ inline Type of_number(float x, int index) { return with(ordered_number(x), index); }
    static __device__ inline uint64_t wide(Type k) {
        if (k <= kOrderedClosed) return 0;
        const uint32_t o = k & 0x80000000u ? k & ~0x1fffu : k | 0x1fffu;
        return (uint64_t)o << 32 | (0xffffffffu - (0x1fffu - (k & 0x1fffu)));
    }
};
template <>
struct RowKey<__bf16> : ShortRowKey {};
template <>
struct RowKey<_Float16> : ShortRowKey {};

__device__ inline uint32_t larger_key(uint32_t a, uint32_t b) { return max(a, b); }
__device__ inline uint64_t larger_key(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ inline uint32_t smaller_key(uint32_t a, uint32_t b) { return min(a, b); }
__device__ inline uint64_t smaller_key(uint64_t a, uint64_t b) { return a < b ? a : b; }

template <int kCtrl>
__device__ inline uint32_t dpp_move_key(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, false);
}
template <int kCtrl>
__device__ inline uint64_t dpp_move_key(uint64_t v) {
    return (uint64_t)dpp_move_key<kCtrl>((uint32_t)(v >> 32)) << 32 | dpp_move_key<kCtrl>((uint32_t)v);
}

// The smallest number of 8 or 16 lanes.
template <int kGroup, typename Key>
__device__ inline Key smallest_of_lanes(Key v) {
    v = smaller_key(v, dpp_move_key<0xb1>(v));
    v = smaller_key(v, dpp_move_key<0x4e>(v));
    v = smaller_key(v, dpp_move_key<0x141>(v));
    if constexpr (kGroup == 16) v = smaller_key(v, dpp_move_key<0x140>(v));
    return v;
}

__device__ inline uint32_t key_of_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ inline uint64_t key_of_lane(uint64_t v, int lane) {
    return (uint64_t)key_of_lane((uint32_t)(v >> 32), lane) << 32 | key_of_lane((uint32_t)v, lane);
}

// Sums of two values, and a maximum, over a group.
template <int kGroup>
__device__ inline float sum_of_lanes(float v) {
    if constexpr (kGroup == 8) {
        v += dpp_move<0xb1, 0xf>(v);
        v += dpp_move<0x4e, 0xf>(v);
        return v + dpp_move<0x141, 0xf>(v);
    } else {
        return sum_of_group<kGroup>(v, nullptr);
    }
}
template <int kGroup>
__device__ inline float2 sums_of_group(float2 v, float2* s_wave) {
    if constexpr (kGroup <= 64) return make_float2(sum_of_lanes<kGroup>(v.x), sum_of_lanes<kGroup>(v.y));
    v = make_float2(wave_reduce_sum(v.x), wave_reduce_sum(v.y));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x / 64] = v;
    __syncthreads();
    v = s_wave[0];
#pragma unroll
    for (int w = 1; w < kGroup / 64; ++w) {
        v.x += s_wave[w].x;
        v.y += s_wave[w].y;
    }
    return v;
}
template <int kGroup>
__device__ inline float largest_of_group(float v, float* s_wave) {
    if constexpr (kGroup == 8) {
        v = fmaxf(v, dpp_move<0xb1, 0xf>(v));
        v = fmaxf(v, dpp_move<0x4e, 0xf>(v));
        return fmaxf(v, dpp_move<0x141, 0xf>(v));
    } else {
        return max_of_group<kGroup>(v, s_wave);
    }
}

// The largest number that at least k of a wave's 64 * kN keys reach, or a lower one that exactly k of them do: its bits are found
// from the highest on, down to kLast (the rest of them 0). 0 if there are fewer keys that are not 0.
template <int kN, int kLast = 0, typename Key>
__device__ inline Key reached_by(const Key (&v)[kN], int k) {
    Key t = 0;
    for (int bit = 8 * (int)sizeof(Key) - 1; bit >= kLast; --bit) {
        const Key up = t | (Key)1 << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < kN; ++i) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= up));
        if (count >= k) t = up;
        if (count == k) break;
    }
    return t;
}

constexpr int kCandidates = 1024;    // of a workgroup's row
constexpr int kManyCandidates = 160;  // from here on the k-th of them is searched before they are ranked

// Keys (LDS) in order: emit(place, key) for the first `top`, 0 where there are fewer. Every key counts those before it.
template <int kGroup, typename Key, typename Emit>
__device__ inline void emit_ranked(const Key* s_keys, int count, int top, int tid, Emit emit) {
    for (int c = tid; c < count; c += kGroup) {
        const Key key = s_keys[c];
        int place = 0;
        for (int j = 0; j < count; ++j) place += s_keys[j] > key ? 1 : 0;
        if (place < top) emit(place, key);
    }
    for (int c = count + tid; c < top; c += kGroup) emit(c, (Key)0);
}

// A wave's keys that are `least` or more (least > 0), together in LDS, at most kMost of them; how many there are.
template <int kN, int kMost, typename Key>
__device__ inline int collect_keys(const Key (&v)[kN], Key least, Key* s_keys, int lane) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const bool mine = v[i] >= least;
        const uint64_t all = __builtin_amdgcn_ballot_w64(mine);
        const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        if (mine && at < kMost) s_keys[at] = v[i];
        count += __builtin_popcountll(all);
    }
    return count;
}

// Of `count` keys in LDS (at most kMost) the first `top`, in no order, by one wave: how many are left.
template <int kMost, typename Key>
__device__ inline int keep_first(Key* s_keys, int count, int top, int lane) {
    if (count <= 64 || count <= top) return count;
    Key v[kMost / 64];
#pragma unroll
    for (int i = 0; i < kMost / 64; ++i) v[i] = i * 64 + lane < count ? s_keys[i * 64 + lane] : 0;
    wave_lds_sync();
    const Key least = reached_by<kMost / 64>(v, top);
    return collect_keys<kMost / 64, kMost>(v, least, s_keys, lane);
}
template <typename Key>
__device__ inline int keep_first_of_any(Key* s_keys, int count, int top, int lane) {
    return count <= 256 ? keep_first<256>(s_keys, count, top, lane) : keep_first<kCandidates>(s_keys, count, top, lane);
}

template <int kGroup>
struct TopScratch {
    uint64_t keys[kCandidates];
    uint32_t most[kGroup];
    uint32_t threshold;
    int count, counts[2];
};

// A row's (or slice's) alternatives by a workgroup. `mine` is the thread's largest logit: what k of them reach is reached by at least
// k logits, so only threads whose own reach it have candidates. Their logits are read again, by their waves. For up to 16
// alternatives the largest of four threads stand for them, which every wave searches for itself (4096 x 65537 with 8: 135 us; each
// wave's own k-th largest, the highest of which bounds the row, let in more: 194); for more one wave searches all. special: there are
// NaN or +inf.
template <typename T, int kGroup, int kVecs, typename Emit>
__device__ inline void top_of_workgroup(const T* __restrict__ z, int64_t length, int64_t from, const Stretch& st, float mine,
                                        float last, bool special, int top, TopScratch<kGroup>& s, Emit emit) {
    constexpr int kElements = Words<T>::kElements;
    const int tid = threadIdx.x, lane = tid & 63;
    __syncthreads();  // the row before is done
    if (tid == 0) {
        s.count = 0;
        s.counts[0] = 0;
        s.counts[1] = 0;
    }
    const uint32_t most = ordered_bits(mine);
    const bool few = top <= kGroup / 16 && top <= 16;
    if (few) {
        uint32_t quad = max(most, dpp_move_key<0xb1>(most));
        quad = max(quad, dpp_move_key<0x4e>(quad));
        if (lane % 4 == 0) s.most[tid / 4] = quad;
    } else {
        s.most[tid] = most;
    }
    __syncthreads();
    if (!special) {
        uint32_t threshold;
        if (few) {
            uint32_t v[kGroup / 256];
#pragma unroll
            for (int i = 0; i < kGroup / 256; ++i) v[i] = s.most[i * 64 + lane];
            threshold = reached_by<kGroup / 256, 16>(v, top);
        } else {
            if (tid < 64) {
                uint32_t v[kGroup / 64];
#pragma unroll
                for (int i = 0; i < kGroup / 64; ++i) v[i] = s.most[i * 64 + tid];
                const uint32_t t = reached_by<kGroup / 64, 16>(v, top);
                if (tid == 0) s.threshold = t;
            }
            __syncthreads();
            threshold = s.threshold;
        }
        const uint32_t least = max(threshold, kOrderedClosed + 1);  // closed logits are no alternatives
        const auto take = [&](float x, int64_t index) {
            if (ordered_bits(x) < least) return;
            const int at = atomicAdd(&s.count, 1);
            if (at < kCandidates) s.keys[at] = key_of(x, from + index);
        };
        // the logits of as many owners together as a wave has lanes for
        constexpr int kHeld = kVecs * kElements, kOwners = kHeld >= 64 ? 1 : 64 / kHeld, kSteps = kHeld >= 64 ? kHeld / 64 : 1;
        for (uint64_t hits = __builtin_amdgcn_ballot_w64(most >= least); hits != 0;) {
            int owner = -1;
#pragma unroll
            for (int o = 0; o < kOwners; ++o) {
                if (hits != 0 && lane / (64 / kOwners) == o) owner = (tid & ~63) + __builtin_ctzll(hits);
                hits &= hits - 1;
            }
            float x[kSteps];
            int64_t at[kSteps];
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
                const int i = u * 64 + lane % (64 / kOwners), vec = i / kElements * kGroup + owner;
                const bool some = owner >= 0 && vec < st.vecs;
                at[u] = some ? st.lead + (int64_t)vec * kElements + i % kElements : -1;
                x[u] = some ? to_float(z[at[u]]) : -INFINITY;  // which is no alternative
            }
#pragma unroll
            for (int u = 0; u < kSteps; ++u) take(x[u], at[u]);
        }
        if (st.loose >= 0) take(last, st.loose);
        __syncthreads();
        int count = s.count;
        if (count <= kCandidates) {
            if (count > kManyCandidates) {
                __syncthreads();  // everybody has read s.count
                if (tid < 64) {
                    const int left = keep_first_of_any(s.keys, count, top, lane);
                    if (tid == 0) s.count = left;
                }
                __syncthreads();
                count = s.count;
            }
            emit_ranked<kGroup>(s.keys, count, top, tid, emit);
            return;
        }
    }
    // More than kCandidates logits at the bound (rows of equal logits, as of a head of zeros, or saturated ones), or some that are not
    // finite: the value of the last alternative is found bit by bit, then the last index that has it. Each count is one more look at
    // the row, 65 in all, one logit a load: all logits equal, in bf16, one row of 131072 with 20 alternatives 268 us (37 of a call
    // otherwise), 200 x 20000 with 8 773 (26), 20000 x 5000 with 20 3400 (110), 4096 x 65537 with 8 22100 (133).
    int turn = 0;
    const auto counted = [&](auto belongs) {
        int n = 0;
        for (int64_t i = tid; i < length; i += kGroup) n += belongs(ordered_bits(to_float(z[i])), (uint32_t)i) ? 1 : 0;
        for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
        if (lane == 0) atomicAdd(&s.counts[turn], n);
        __syncthreads();
        n = s.counts[turn];
        turn ^= 1;
        if (tid == 0) s.counts[turn] = 0;
        __syncthreads();
        return n;
    };
    const int open = counted([](uint32_t o, uint32_t) { return o > kOrderedClosed; }), need = min(top, open);
    uint32_t value = 0, end = 0;
    if (need > 0) {
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t up = value | 1u << bit;
            if (counted([&](uint32_t o, uint32_t) { return o >= up; }) >= need) value = up;
        }
        const int equal = need - counted([&](uint32_t o, uint32_t) { return o > value; });
        for (int bit = 30; bit >= 0; --bit) {  // as many indices lie below `end` as leave less than `equal` before it
            const uint32_t up = end + (1u << bit);
            if (counted([&](uint32_t o, uint32_t i) { return o == value && i < up; }) < equal) end = up;
        }
    }
    if (tid == 0) s.count = 0;
    __syncthreads();
    for (int64_t i = tid; need > 0 && i < length; i += kGroup) {
        const float x = to_float(z[i]);
        const uint32_t o = ordered_bits(x);
        if (o > value || (o == value && (uint32_t)i <= end)) s.keys[atomicAdd(&s.count, 1)] = key_of(x, from + i);
    }
    __syncthreads();
    emit_ranked<kGroup>(s.keys, need, top, tid, emit);
}

// What a row's sums say to the outside.
struct RowAnswer {
    float m, log_s, inv_t;
    __device__ inline float log_q(float z) const {
        return z == -INFINITY && log_s == log_s ? -INFINITY : (z - m) * inv_t - log_s;
    }
};
__device__ inline RowAnswer answer_of(const LogProbsArgs& a, RowSums q) { return {q.m, logf(q.s), a.inv_t}; }
__device__ inline float entropy_of(RowSums q) { return q.s == 0.0f ? 0.0f : logf(q.s) - kLn2 * (q.w / q.s); }

__device__ inline int32_t id_of(const LogProbsArgs& a, int64_t row) { return a.ids != nullptr ? a.ids[row] : -1; }

// A row's given label and its logit, two loads of which the second waits for the first. Groups of 8 and 16 lanes ask for them
// beside the row (307200 x 150 with the gradient 58 us, 62 at the row's end, with vectors of eight logits), larger ones, whose other
// waves go on meanwhile, at its end (100000 x 1000 in bf16 by a wave a row 65 us, beside the row 71).
struct GivenLabel {
    int32_t id;
    bool known;
    float z;
};
template <typename T>
__device__ inline GivenLabel given_label(const LogProbsArgs& a, int64_t row, const T* __restrict__ z) {
    GivenLabel g;
    g.id = id_of(a, row);
    g.known = g.id >= 0 && g.id < a.vocab;
    g.z = g.known ? to_float(z[g.id]) : 0.0f;
    return g;
}

// By one thread: a row's chosen log probability, entropy and statistics.
__device__ inline void write_row(const LogProbsArgs& a, int64_t row, const GivenLabel& given, RowSums q) {
    if (a.chosen != nullptr) a.chosen[row] = given.known ? answer_of(a, q).log_q(given.z) : 0.0f;
    const float h = entropy_of(q);
    if (a.entropy != nullptr) a.entropy[row] = h;
    if (a.stats != nullptr) {
        a.stats[3 * row] = q.m;
        a.stats[3 * row + 1] = q.s;
        a.stats[3 * row + 2] = h;
    }
}

__device__ inline void write_alternative(const LogProbsArgs& a, int64_t row, int place, uint64_t key, RowAnswer r) {
    const int64_t at = row * a.top + place;
    a.top_ids[at] = key == 0 ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
    a.top_logs[at] = key == 0 ? -INFINITY : r.log_q(ordered_value((uint32_t)(key >> 32)));
}

// A row's gradient: dz = e (rate + slope u), and `own` more at the given label.
struct RowGrad {
    bool live;
    float base, rate, slope, own;
    int32_t id;
    __device__ inline float of(float z, float e, float scale2, bool sloped) const {
        return sloped ? e * __builtin_fmaf(slope, fmaxf((z - base) * scale2, kLeastExponent2), rate) : e * rate;
    }
    __device__ inline float at(float z, float scale2, bool sloped) const {
        return of(z, __builtin_amdgcn_exp2f((z - base) * scale2), scale2, sloped);
    }
};
__device__ inline RowGrad grad_of(const LogProbsArgs& a, int64_t row, int32_t id, float m, float s, float h) {
    RowGrad g;
    const bool known = id >= 0 && id < a.vocab;
    g.id = id;
    const float gl = known ? a.grad_scale * (a.row_grad != nullptr ? a.row_grad[row] : 1.0f) : 0.0f;
    const float gh = a.entropy_scale * (a.entropy_grad != nullptr ? a.entropy_grad[row] : 1.0f);
    g.live = (gl != 0.0f || gh != 0.0f) && s != 0.0f;
    g.base = m == -INFINITY ? 0.0f : m;
    const float over = g.live ? a.inv_t / s : 0.0f;
    g.slope = -(gh * kLn2) * over;
    g.rate = -(gl + gh * (h - logf(s))) * over;
    g.own = gl * a.inv_t;
    if (!known) g.id = -1;
    return g;
}

// Rows that fit the registers of a group: kGroup threads hold kVecs vectors of 16 bytes each. Groups of 8 lanes take vectors of four
// logits, so that fewer lanes stand idle at the row's end (307200 x 150 with the gradient and three alternatives: in bf16 62 us, 70
// with eight logits; in float32 88, 106 by groups of 16), from the row's start on, at whatever address that is, and at most one
// logit a thread behind the last vector.
template <typename T, int kGroup, int kVecs>
struct HeldRow {
    static constexpr int kWords = kGroup == 8 ? (int)sizeof(T) : 4, kElements = Words<T, kWords>::kElements;
    static constexpr bool kKeeps = kGroup == 8;  // what sums() computes, for a gradient of the same pass
    Words<T, kWords> x[kVecs];
    float e[kKeeps ? kVecs * kElements : 1];
    float last;
    Stretch st;

    __device__ inline void load(const T* __restrict__ z, int64_t length, int tid) {
        if constexpr (kGroup == 8) {
            st.lead = 0;
            st.vecs = (int)length / kElements;
            st.loose = st.vecs * kElements + tid < length ? st.vecs * kElements + tid : -1;
        } else {
            st = stretch_of<T>(z, length, tid);
        }
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
            x[u] = load_words<T, kWords>(z + st.lead + u * kGroup * kElements, tid, st.vecs - u * kGroup);
        last = st.loose >= 0 ? to_float(z[st.loose]) : -INFINITY;
    }
    __device__ inline float largest() const {
        float m = last == last ? last : -INFINITY;
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
            for (int i = 0; i < kElements; ++i) m = fmaxf(m, element_of(x[u], i));
        return m;
    }
    __device__ inline float2 sums(float base, float scale2) {
        float2 r;
        r.x = __builtin_amdgcn_exp2f((last - base) * scale2);
        r.y = r.x * scaled_from(last, base, scale2);
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            repack(x[u]);
#pragma unroll
            for (int i = 0; i < kElements; ++i) {
                const float v = (element_of(x[u], i) - base) * scale2;
                const float power = __builtin_amdgcn_exp2f(v);
                r.x += power;
                r.y = __builtin_fmaf(power, fmaxf(v, kLeastExponent2), r.y);
                if constexpr (kKeeps) e[u * kElements + i] = power;
            }
            asm volatile("" : "+v"(r.x), "+v"(r.y));  // both sums go on with each vector: no e is kept for later
        }
        return r;
    }
};

// A row's alternatives by a wave, from the registers that hold the row. `mine` is the lane's largest logit: what `top` lanes' reach
// is reached by at least `top` logits, so all others are none. (16 bits of that bound are enough: a lower one lets in a few more.)
// The candidates come together in LDS, thinned out where they are many, and the last 64 of them are ranked lane against lane.
// special: there are NaN or +inf, the row is read again.
template <typename T>
constexpr int kWaveCandidates = 64 * Words<T>::kElements + 128;  // what is left of the ones before, and all of a vector

template <typename T, int kVecs, typename Emit>
__device__ inline void top_of_wave(const T* __restrict__ z, int vocab, HeldRow<T, 64, kVecs>& x, float mine, bool special, int top,
                                   int lane, typename RowKey<T>::Type* s_keys, Emit emit) {
    typedef typename RowKey<T>::Type Key;
    constexpr int kElements = Words<T>::kElements, kFew = 4;
    int count = 0;
    wave_lds_sync();  // the row before is done
    const auto put = [&](bool in, uint64_t all, float v, int index) {
        const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        if (in) s_keys[at] = RowKey<T>::of(v, index);
        count += __builtin_popcountll(all);
    };
    const auto thin = [&] {
        wave_lds_sync();
        if (count <= 128) count = keep_first<128>(s_keys, count, top, lane);
        else count = keep_first<kWaveCandidates<T>>(s_keys, count, top, lane);
        wave_lds_sync();
    };
    if (vocab <= 64 * kFew) {  // few lanes hold the row: every lane takes some of it again
        Key v[kFew];
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            const int at = i * 64 + lane;
            v[i] = at < vocab ? RowKey<T>::of(to_float(z[at]), at) : (Key)0;
            if (v[i] <= RowKey<T>::of(-INFINITY, 0)) v[i] = 0;
        }
        const Key least = reached_by<kFew>(v, top);
        count = collect_keys<kFew, kWaveCandidates<T>>(v, least > 0 ? least : (Key)1, s_keys, lane);
    } else if (!special) {
        const uint32_t most[1] = {ordered_bits(mine)};
        const float bound = ordered_value(max(reached_by<1, 16>(most, top), kOrderedClosed + 1));
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            if (count > 128) thin();
            repack(x.x[u]);
#pragma unroll
            for (int i = 0; i < kElements; ++i) {
                const float v = element_of(x.x[u], i);
                const bool in = v >= bound;
                const uint64_t all = __builtin_amdgcn_ballot_w64(in);
                if (all != 0) put(in, all, v, x.st.lead + (u * 64 + lane) * kElements + i);
            }
        }
        const bool in = x.st.loose >= 0 && x.last >= bound;
        if (count > 128) thin();
        put(in, __builtin_amdgcn_ballot_w64(in), x.last, (int)x.st.loose);
    } else {
        for (int i0 = 0; i0 < vocab; i0 += 64) {
            if (count > 128) thin();
            const int at = min(i0 + lane, vocab - 1);
            const float v = to_float(z[at]);
            const bool in = i0 + lane < vocab && v != -INFINITY;
            put(in, __builtin_amdgcn_ballot_w64(in), v, at);
        }
    }
    if (count > 64) thin();
    wave_lds_sync();
    const Key key = lane < count ? s_keys[lane] : 0;
    int place = 0;
    for (int j = 0; j < count; ++j) place += key_of_lane(key, j) > key ? 1 : 0;
    if (lane < count ? place < top : lane < top) emit(lane < count ? place : lane, RowKey<T>::wide(key));
}

// NaN of a word's one or two logits without their signs, which comes before every number.
template <typename T>
__device__ inline uint32_t positive_nans(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return (w & 0x7fffffffu) > 0x7f800000u ? 0x7fffffffu : w;
    } else {
        constexpr uint32_t kInf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
        if ((w & 0x7fffu) > kInf) w = (w | 0x7fffu) & ~0x8000u;
        if ((w >> 16 & 0x7fffu) > kInf) w = (w | 0x7fff0000u) & 0x7fffffffu;
        return w;
    }
}

// What a NaN is then as a number, also one that is not in a vector: equal ones go by their indices.
template <typename T>
__device__ inline float positive_nan() {
    Words<T, 1> x;
    x.w[0] = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
    return element_of(x, 0);
}

// One alternative after the other, from keys in the registers of 8 or 16 lanes: of the keys up to a bound, the nearest. How far a
// key lies below it wraps around for those that do not. Lane p keeps the one at place p until there is one for each lane. special:
// there is NaN in the wave's rows.
template <typename T, int kGroup, int kVecs, typename Emit>
__device__ inline void top_of_lanes(HeldRow<T, kGroup, kVecs>& x, bool special, int top, int tid, Emit emit) {
    typedef typename RowKey<T>::Type Key;
    constexpr int kWords = HeldRow<T, kGroup, kVecs>::kWords, kElements = HeldRow<T, kGroup, kVecs>::kElements;
    constexpr int kKeys = kVecs * kElements + 1;
    Key keys[kKeys];
    if (special) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
            for (int i = 0; i < kWords; ++i) x.x[u].w[i] = positive_nans<T>(x.x[u].w[i]);
        if (x.last != x.last) x.last = positive_nan<T>();
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
        const int vec = u * kGroup + tid;
        repack(x.x[u]);
#pragma unroll
        for (int i = 0; i < kElements; ++i)  // behind the row's end lies -inf
            keys[u * kElements + i] = RowKey<T>::of_number(element_of(x.x[u], i), x.st.lead + vec * kElements + i);
    }
    keys[kKeys - 1] = RowKey<T>::of_number(x.last, max((int)x.st.loose, 0));
    Key most = ~(Key)0, mine = 0;
    for (int first = 0; first < top; first += kGroup) {
        const int count = min(top - first, kGroup);
        for (int place = 0; place < count; ++place) {
            Key apart = most - keys[0];
#pragma unroll
            for (int i = 1; i < kKeys; ++i) apart = smaller_key(apart, most - keys[i]);
            apart = smallest_of_lanes<kGroup>(apart);
            const Key best = most - apart;  // above the bound where none is left
            if (place == tid) mine = best <= most ? best : 0;
            if (best <= most) most = best - 1;
        }
        if (tid < count) emit(first + tid, RowKey<T>::wide(mine));
    }
}

// A row is read once: its largest logit, both sums, the gradient and the alternatives come from registers. Long rows are bound by
// memory (4096 x 65537 in bf16: sums 111 us, 4.8 TB/s; with the gradient 224, 4.8; 8 alternatives more 24 and 17). Short ones are
// bound by the vector units, never idle (307200 x 150 in bf16: sums 27 us, 3.4 TB/s; with the gradient 45, 4.1; three alternatives
// more 14 and 17). Four waves a SIMD at least: 128 registers, of which a row has 64.
template <typename T, int kGroup, int kVecs>
__global__ __launch_bounds__(kGroup < 256 ? 256 : kGroup, 4) void logprobs_held_kernel(LogProbsArgs a,
                                                                                       const T* __restrict__ logits,
                                                                                       T* __restrict__ grad) {
    constexpr int kGroups = kGroup < 256 ? 256 / kGroup : 1;  // rows of a workgroup
    constexpr int kWords = HeldRow<T, kGroup, kVecs>::kWords, kElements = HeldRow<T, kGroup, kVecs>::kElements;
    __shared__ TopScratch<kGroups == 1 ? kGroup : 1> s_top[1];
    __shared__ typename RowKey<T>::Type s_keys[kGroup == 64 ? kGroups : 1][kWaveCandidates<T>];
    __shared__ float2 s_wave2[16];
    __shared__ float s_wave[16];
    const int group = kGroups == 1 ? 0 : threadIdx.x / kGroup, tid = kGroups == 1 ? threadIdx.x : threadIdx.x % kGroup;
    for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < a.rows; row += (int64_t)gridDim.x * kGroups) {
        const T* const z = logits + row * a.logits_stride;
        HeldRow<T, kGroup, kVecs> x;
        x.load(z, a.vocab, tid);
        GivenLabel given;
        if (kGroup < 64) given = given_label(a, row, z);
        const float mine = x.largest();
        RowSums q;
        float h;
        if (kGroup == 8 && a.backward) {
            q.m = a.stats[3 * row];
            q.s = a.stats[3 * row + 1];
            h = a.stats[3 * row + 2];
            x.sums(q.m == -INFINITY ? 0.0f : q.m, a.scale2);
        } else {
            q.m = largest_of_group<kGroup>(mine, s_wave);
            const float base = q.m == -INFINITY ? 0.0f : q.m;
            const float2 sums = sums_of_group<kGroup>(x.sums(base, a.scale2), s_wave2);
            q.s = sums.x;
            q.w = sums.y;
            h = entropy_of(q);
        }
        if (tid == 0 && !(kGroup == 8 && a.backward)) {
            if (kGroup >= 64) given = given_label(a, row, z);
            write_row(a, row, given, q);
        }
        if (grad != nullptr) {
            T* const g = grad + row * a.grad_stride;
            const RowGrad d = grad_of(a, row, kGroup < 64 ? given.id : id_of(a, row), q.m, q.s, h);
            const bool sloped = d.slope != 0.0f;
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                float y[kElements];
                repack(x.x[u]);
#pragma unroll
                for (int i = 0; i < kElements; ++i) {
                    const float v = element_of(x.x[u], i);
                    if constexpr (HeldRow<T, kGroup, kVecs>::kKeeps)
                        y[i] = d.live ? d.of(v, x.e[u * kElements + i], a.scale2, sloped) : 0.0f;
                    else
                        y[i] = d.live ? d.at(v, a.scale2, sloped) : 0.0f;
                }
                const int own = d.id - x.st.lead - (u * kGroup + tid) * kElements;
                if (d.live && d.id >= 0 && own >= 0 && own < kElements) {
#pragma unroll
                    for (int i = 0; i < kElements; ++i) y[i] += i == own ? d.own : 0.0f;
                }
                store_words<T, kWords, kWords == 4>(g + x.st.lead + u * kGroup * kElements, tid, x.st.vecs - u * kGroup, y);
            }
            if (x.st.loose >= 0)
                g[x.st.loose] =
                    from_float<T>(d.live ? d.at(x.last, a.scale2, sloped) + (d.id == x.st.loose ? d.own : 0.0f) : 0.0f);
        }
        if (a.top == 0) continue;
        const RowAnswer r = answer_of(a, q);
        const auto emit = [&](int place, uint64_t key) { write_alternative(a, row, place, key, r); };
        if constexpr (kGroup < 64)
            top_of_lanes<T, kGroup, kVecs>(x, __builtin_amdgcn_ballot_w64(q.s != q.s) != 0, a.top, tid, emit);
        else if constexpr (kGroup == 64)
            top_of_wave<T, kVecs>(z, (int)a.vocab, x, mine, q.s != q.s, a.top, tid, s_keys[group], emit);
        else top_of_workgroup<T, kGroup, kVecs>(z, a.vocab, 0, x.st, mine, x.last, q.s != q.s, a.top, s_top[0], emit);
    }
}

// Longer rows, and few of them: a row is cut into slices, each held by a workgroup. This launch leaves every slice's sums and its
// first alternatives,
constexpr int kSliceGroup = 256;

template <typename T, int kVecs>
__global__ __launch_bounds__(kSliceGroup) void logprobs_slices_kernel(LogProbsArgs a, const T* __restrict__ logits) {
    __shared__ TopScratch<kSliceGroup> s_top;
    __shared__ float2 s_wave2[16];
    __shared__ float s_wave[16];
    const int64_t total = a.rows * a.slices;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t row = b / a.slices, from = b % a.slices * a.slice, to = min(from + a.slice, a.vocab);
        HeldRow<T, kSliceGroup, kVecs> x;
        x.load(logits + row * a.logits_stride + from, to - from, threadIdx.x);
        const float mine = x.largest();
        const float m = max_of_group<kSliceGroup>(mine, s_wave);
        const float base = m == -INFINITY ? 0.0f : m;
        const float2 sums = sums_of_group<kSliceGroup>(x.sums(base, a.scale2), s_wave2);
        if (threadIdx.x == 0) a.partial[b] = {m, sums.x, sums.y};
        if (a.top > 0)
            top_of_workgroup<T, kSliceGroup, kVecs>(logits + row * a.logits_stride + from, to - from, from, x.st, mine, x.last,
                                                    sums.x != sums.x, a.top, s_top,
                                                    [&](int place, uint64_t key) { a.partial_top[b * a.top + place] = key; });
    }
}

// and this one joins a row's.
template <typename T>
__global__ __launch_bounds__(kSliceGroup) void logprobs_join_kernel(LogProbsArgs a, const T* __restrict__ logits) {
    __shared__ uint64_t s_keys[kCandidates], s_least;
    __shared__ float2 s_wave2[16];
    __shared__ float s_wave[16];
    __shared__ int s_count;
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const RowSums* const part = a.partial + row * a.slices;
        const GivenLabel given = given_label(a, row, logits + row * a.logits_stride);
        const uint64_t* const keys = a.partial_top + row * a.slices * a.top;
        // Of each slice the key at place p, top <= slices (p + 1): those that reach the k-th largest of them, k (p + 1) >= top,
        // come from slices that have enough keys together, so no alternative is below it.
        uint64_t most[1] = {0};
        const int p = a.top > 0 ? (int)((a.top - 1) / a.slices) : 0;
        float m = -INFINITY;
        for (int64_t i = tid; i < a.slices; i += kSliceGroup) {
            m = fmaxf(m, part[i].m);
            if (a.top > 0) most[0] = larger_key(most[0], keys[i * a.top + p]);
        }
        RowSums q;
        q.m = max_of_group<kSliceGroup>(m, s_wave);
        const float base = q.m == -INFINITY ? 0.0f : q.m;
        float2 sums = make_float2(0.0f, 0.0f);
        for (int64_t i = tid; i < a.slices; i += kSliceGroup) {
            const RowSums p = part[i];
            const float u = scaled_from(p.m, base, a.scale2), f = __builtin_amdgcn_exp2f((p.m - base) * a.scale2);
            sums.x += f * p.s;
            sums.y += f * (p.w + u * p.s);
        }
        if (tid == 0) {
            s_count = 0;
            s_least = 0;
        }
        if (a.top > 0) s_keys[tid] = most[0];
        sums = sums_of_group<kSliceGroup>(sums, s_wave2);
        q.s = sums.x;
        q.w = sums.y;
        if (tid == 0) write_row(a, row, given, q);
        if (a.top == 0) continue;
        const RowAnswer r = answer_of(a, q);
        if (tid < 64) {  // by the logits' bits alone
            const int k = (a.top + p) / (p + 1);
            uint64_t v[kSliceGroup / 64];
#pragma unroll
            for (int i = 0; i < kSliceGroup / 64; ++i) v[i] = s_keys[i * 64 + tid];
            uint64_t t;
            if (a.slices <= 64) {
                const uint64_t few[1] = {v[0]};
                t = reached_by<1, 32>(few, k);
            } else {
                t = reached_by<kSliceGroup / 64, 32>(v, k);
            }
            if (tid == 0) s_least = t;
        }
        __syncthreads();
        const int64_t all = a.slices * a.top;
        const uint64_t least = larger_key(s_least, (uint64_t)1);
        for (int64_t i0 = 0; i0 < all; i0 += kSliceGroup) {
            const uint64_t key = i0 + tid < all ? keys[i0 + tid] : 0;
            if (key >= least) s_keys[atomicAdd(&s_count, 1)] = key;
            __syncthreads();
            const int count = s_count;
            __syncthreads();  // everybody has read it
            if (count + kSliceGroup > kCandidates || (i0 + kSliceGroup >= all && count > kManyCandidates)) {
                if (tid < 64) {
                    const int left = keep_first_of_any(s_keys, count, a.top, tid);
                    if (tid == 0) s_count = left;
                }
                __syncthreads();
            }
        }
        emit_ranked<kSliceGroup>(s_keys, s_count, a.top, tid,
                                 [&](int place, uint64_t key) { write_alternative(a, row, place, key, r); });
        __syncthreads();
    }
}

// The gradient from a forward's statistics: kGroup threads take a stretch of a row. Bound by memory (4096 x 65537 in bf16 184 us, 5.8
// TB/s; 307200 x 150 in float32 74, 5.0).
template <typename T, int kGroup>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogProbsArgs a, const T* __restrict__ logits,
                                                            T* __restrict__ grad) {
    constexpr int kGroups = 256 / kGroup, kElements = Words<T>::kElements, kAhead = 4;
    const int group = threadIdx.x / kGroup, tid = threadIdx.x % kGroup;
    const int64_t total = a.rows * a.slices;
    for (int64_t b = (int64_t)blockIdx.x * kGroups + group; b < total; b += (int64_t)gridDim.x * kGroups) {
        const int64_t row = b / a.slices, from = b % a.slices * a.slice, to = min(from + a.slice, a.vocab);
        const T* const z = logits + row * a.logits_stride + from;
        T* const g = grad + row * a.grad_stride + from;
        const RowGrad d = grad_of(a, row, id_of(a, row), a.stats[3 * row], a.stats[3 * row + 1], a.stats[3 * row + 2]);
        const bool sloped = d.slope != 0.0f;
        const Stretch st = stretch_of<T>(z, to - from, tid);
        for (int v = tid; v < st.vecs; v += kGroup * kAhead) {
            Words<T> x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) x[u] = load_words<T>(z + st.lead, v + u * kGroup, d.live ? st.vecs : 0);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (v + u * kGroup >= st.vecs) continue;
                float y[kElements];
#pragma unroll
                for (int i = 0; i < kElements; ++i) y[i] = d.live ? d.at(element_of(x[u], i), a.scale2, sloped) : 0.0f;
                const int64_t own = d.id - from - st.lead - (int64_t)(v + u * kGroup) * kElements;
                if (d.live && d.id >= 0 && own >= 0 && own < kElements) {
#pragma unroll
                    for (int i = 0; i < kElements; ++i) y[i] += i == own ? d.own : 0.0f;
                }
                store_words<T>(g + st.lead, v + u * kGroup, st.vecs, y);
            }
        }
        if (st.loose >= 0)
            g[st.loose] = from_float<T>(
                d.live ? d.at(to_float(z[st.loose]), a.scale2, sloped) + (d.id >= 0 && d.id - from == st.loose ? d.own : 0.0f) : 0.0f);
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

// How a forward goes: by groups that hold whole rows (group > 0), or by slices. The smallest group that holds a row, in vectors as
// many as its kernels have, or 16 above 16 KB, where there are rows enough for the GPU's 256 CUs (4096 x 65537 with 8 alternatives
// 135 us, in slices 189 to 213; one row of 131072 15 us in slices). Rows of 8 lanes whatever the alternatives are (307200 x 150 in
// bf16 with 20 of them 88 us, a wave a row 290; 100000 x 180 in float32 with 64, the worst, 197); of 16 lanes up to 16 of them, or 8
// in float32 and of more than 64 vectors (100000 x 1000 with 5 of them 87 us, with 16 130; a wave a row 105 and 118; 252716 x 565
// with 3 104 and 238).
struct LogProbsPlan {
    int group, vecs;
    int64_t slice, slices;
};

LogProbsPlan logprobs_plan(int64_t rows, int64_t vocab, int64_t bytes, int32_t top) {
    LogProbsPlan p = {};
    const int64_t vecs = vocab * bytes / 16;
    if (vocab / 4 <= 8 * (bytes == 4 ? 6 : 8)) {
        p.group = 8;
        p.vecs = vocab >= 4 ? (int)ceil_div(vocab / 4, 8) : 1;
        return p;
    }
    if (vecs <= 16 * (bytes == 4 ? 6 : 8) && top <= (bytes == 4 || vecs > 64 ? 8 : 16)) p.group = 16;
    else if (vecs <= 64 * 4) p.group = 64;
    else if (vecs <= 256 * 4 || (vecs <= 256 * 16 && rows >= 192)) p.group = 256;
    else if (vecs <= 512 * 16 && rows >= 192) p.group = 512;
    else if (vecs <= 1024 * 16 && rows >= 192) p.group = 1024;
    if (p.group != 0) {
        p.vecs = vecs > 0 ? (int)ceil_div(vecs, p.group) : 1;
        return p;
    }
    // slices of 16 KB, or of 64 KB where that makes 1024 of them
    const int64_t most = 65536 / bytes, least = 16384 / bytes;
    p.slice = rows * ceil_div(vocab, most) >= 1024 ? most : least;
    p.vecs = p.slice == most ? 16 : 4;
    p.slices = ceil_div(vocab, p.slice);
    return p;
}

int64_t sums_bytes(int64_t rows, int64_t slices) { return ceil_div(rows * slices * (int64_t)sizeof(RowSums), 16) * 16; }

inline dim3 logprobs_grid(int64_t blocks) { return dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)); }

template <typename T, int kGroup, int kVecs>
gsx_hip_status launch_held(const LogProbsArgs& a, const T* logits, T* grad, hipStream_t stream) {
    const int per = kGroup < 256 ? 256 / kGroup : 1;
    hipLaunchKernelGGL((logprobs_held_kernel<T, kGroup, kVecs>), logprobs_grid(ceil_div(a.rows, per)),
                       dim3(kGroup < 256 ? 256 : kGroup), 0, stream, a, logits, grad);
    return fields_launched("log probabilities launch");
}

// Rows of 8 lanes.
template <typename T>
gsx_hip_status launch_short(int vecs, const LogProbsArgs& a, const T* logits, T* grad, hipStream_t stream) {
    if (vecs <= 1) return launch_held<T, 8, 1>(a, logits, grad, stream);
    if (vecs <= 2) return launch_held<T, 8, 2>(a, logits, grad, stream);
    if (vecs <= 3) return launch_held<T, 8, 3>(a, logits, grad, stream);
    if (vecs <= 4) return launch_held<T, 8, 4>(a, logits, grad, stream);
    if (vecs <= 5) return launch_held<T, 8, 5>(a, logits, grad, stream);
    if constexpr (sizeof(T) == 4) {
        return launch_held<T, 8, 6>(a, logits, grad, stream);
    } else {
        if (vecs <= 6) return launch_held<T, 8, 6>(a, logits, grad, stream);
        return launch_held<T, 8, 8>(a, logits, grad, stream);
    }
}

template <typename T>
gsx_hip_status launch_grad(LogProbsArgs a, const T* logits, T* grad, hipStream_t stream) {
    // rows that 8 lanes hold, in 16 bits, as in the forward: 307200 x 150 43 us, through the other kernel 54; in float32 102 and 74
    const LogProbsPlan p = logprobs_plan(a.rows, a.vocab, sizeof(T), 0);
    if (sizeof(T) == 2 && p.group == 8) {
        a.backward = true;
        a.top = 0;
        return launch_short<T>(p.vecs, a, logits, grad, stream);
    }
    const int64_t vecs = a.vocab * (int64_t)sizeof(T) / 16;
    const auto go = [&](auto kernel, int groups) {
        hipLaunchKernelGGL(kernel, logprobs_grid(ceil_div(a.rows * a.slices, groups)), dim3(256), 0, stream, a, logits, grad);
    };
    a.slice = a.vocab;
    a.slices = 1;
    if (vecs <= 96) go(logprobs_grad_kernel<T, 16>, 16);  // 252716 x 565 in bf16 140 us, by 64 lanes 196; 100000 x 1000 78 and 74
    else if (vecs <= 256) go(logprobs_grad_kernel<T, 64>, 4);
    else {
        a.slice = 16384 / (int64_t)sizeof(T);
        a.slices = ceil_div(a.vocab, a.slice);
        go(logprobs_grad_kernel<T, 256>, 1);
    }
    return fields_launched("log probabilities launch");
}

template <typename T>
gsx_hip_status launch_logprobs(const LogProbsPlan& p, LogProbsArgs a, const T* logits, T* grad, void* temp,
                               hipStream_t stream) {
    if (p.group == 8) return launch_short<T>(p.vecs, a, logits, grad, stream);
    if (p.group == 16) {
        if constexpr (sizeof(T) == 2)
            if (p.vecs <= 3) return launch_held<T, 16, 3>(a, logits, grad, stream);
        if (p.vecs <= 4) return launch_held<T, 16, 4>(a, logits, grad, stream);
        if (p.vecs <= 5) return launch_held<T, 16, 5>(a, logits, grad, stream);
        if constexpr (sizeof(T) == 4) {
            return launch_held<T, 16, 6>(a, logits, grad, stream);
        } else {
            if (p.vecs <= 6) return launch_held<T, 16, 6>(a, logits, grad, stream);
            return launch_held<T, 16, 8>(a, logits, grad, stream);
        }
    }
    if (p.group == 64) {
        if (p.vecs <= 1) return launch_held<T, 64, 1>(a, logits, grad, stream);
        return launch_held<T, 64, 4>(a, logits, grad, stream);
    }
    if (p.group == 256) {
        if (p.vecs <= 4) return launch_held<T, 256, 4>(a, logits, grad, stream);
        if (p.vecs <= 8) return launch_held<T, 256, 8>(a, logits, grad, stream);
        return launch_held<T, 256, 16>(a, logits, grad, stream);
    }
    if (p.group == 512) return launch_held<T, 512, 16>(a, logits, grad, stream);
    if (p.group == 1024) return launch_held<T, 1024, 16>(a, logits, grad, stream);
    a.slice = p.slice;
    a.slices = p.slices;
    a.partial = static_cast<RowSums*>(temp);
    a.partial_top = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(temp) + sums_bytes(a.rows, p.slices));
    const dim3 grid = logprobs_grid(a.rows * p.slices);
    if (p.vecs == 16) hipLaunchKernelGGL((logprobs_slices_kernel<T, 16>), grid, dim3(kSliceGroup), 0, stream, a, logits);
    else hipLaunchKernelGGL((logprobs_slices_kernel<T, 4>), grid, dim3(kSliceGroup), 0, stream, a, logits);
    hipLaunchKernelGGL((logprobs_join_kernel<T>), logprobs_grid(a.rows), dim3(kSliceGroup), 0, stream, a, logits);
    if (grad == nullptr) return fields_launched("log probabilities launch");
    return launch_grad<T>(a, logits, grad, stream);
}

gsx_hip_status logprobs_check(const LogProbsArgs& a, const void* logits, int32_t type, float temperature, const void* grad) {
    if (!known_type(type)) return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "log probabilities: logits are f32, bf16 or f16");
    if (a.vocab < 1 || a.vocab > INT32_MAX)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "log probabilities: 1 to 2^31 - 1 logits a row");
    if (a.top < 0 || a.top > kMostAlternatives || a.top > a.vocab)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "log probabilities: 0 to 64 alternatives, no more than logits");
    if (!rows_fit(a.rows, a.logits_stride, a.vocab) ||
        (grad != nullptr && !rows_fit(a.rows, a.grad_stride, a.vocab)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "log probabilities: rows must be >= 0 and strides at least the row's length");
    if (!(temperature >= 1e-6f) || !(temperature <= 1e6f))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities: the temperature must lie between 1e-6 and 1e6");
    if (a.rows > 0 && (logits == nullptr || (a.top > 0 && (a.top_ids == nullptr || a.top_logs == nullptr))))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities: null pointer");
    if (!aligned_to(logits, type_bytes(type)) || !aligned_to(grad, type_bytes(type)) || !aligned_to(a.ids, 4) ||
        !aligned_to(a.chosen, 4) || !aligned_to(a.entropy, 4) || !aligned_to(a.stats, 4) || !aligned_to(a.top_ids, 4) ||
        !aligned_to(a.top_logs, 4) || !aligned_to(a.row_grad, 4) || !aligned_to(a.entropy_grad, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities: pointers must be aligned to their elements");
    if (logits != nullptr && logits == grad)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities: the gradient may not overwrite the logits");
    return GSX_HIP_SUCCESS;
}

LogProbsArgs logprobs_args(int64_t logits_stride, int64_t rows, int64_t vocab, const int32_t* ids, float temperature,
                           const float* row_grad, float grad_scale, const float* entropy_grad, float entropy_scale,
                           int64_t grad_stride) {
    LogProbsArgs a = {};
    a.rows = rows;
    a.vocab = vocab;
    a.logits_stride = logits_stride;
    a.grad_stride = grad_stride;
    a.ids = ids;
    a.inv_t = 1.0f / temperature;
    a.scale2 = kLog2e / temperature;
    a.row_grad = row_grad;
    a.grad_scale = grad_scale;
    a.entropy_grad = entropy_grad;
    a.entropy_scale = entropy_scale;
    return a;
}

}  // namespace

extern "C" {

size_t gsx_hip_log_probs_temp_bytes(int64_t rows, int64_t vocab, int32_t top) {
    if (rows <= 0 || vocab <= 0 || vocab > INT32_MAX || top < 0 || top > kMostAlternatives || rows > (INT64_MAX >> 4) / vocab)
        return 0;
    int64_t most = 0;  // whatever the logits' type is
    for (int64_t bytes = 2; bytes <= 4; bytes += 2) {
        const LogProbsPlan p = logprobs_plan(rows, vocab, bytes, top);
        if (p.group != 0) continue;
        const int64_t need = sums_bytes(rows, p.slices) + rows * p.slices * top * 8;
        if (need > most) most = need;
    }
    return (size_t)most;
}

gsx_hip_status gsx_hip_log_probs_forward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                         int64_t vocab, const int32_t* ids, float temperature, float* chosen,
                                         float* entropy, float* row_stats, int32_t top, int32_t* top_ids,
                                         float* top_log_probs, void* grad_logits, int64_t grad_stride,
                                         const float* row_grad, float grad_scale, const float* entropy_grad,
                                         float entropy_scale, void* temp, hipStream_t stream) {
    LogProbsArgs a = logprobs_args(logits_stride, rows, vocab, ids, temperature, row_grad, grad_scale, entropy_grad,
                                   entropy_scale, grad_stride);
    a.chosen = chosen;
    a.entropy = entropy;
    a.stats = row_stats;
    a.top = top;
    a.top_ids = top_ids;
    a.top_logs = top_log_probs;
    const gsx_hip_status st = logprobs_check(a, logits, logits_type, temperature, grad_logits);
    if (st != GSX_HIP_SUCCESS || rows == 0) return st;
    const LogProbsPlan p = logprobs_plan(rows, vocab, type_bytes(logits_type), top);
    if (p.group == 0 && (temp == nullptr || !aligned_to(temp, 16)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "log probabilities: the workspace must be non-null and 16-byte aligned");
    if (grad_logits != nullptr && row_stats == nullptr)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities: a gradient needs row_stats");
    return with_type(logits_type, [&](auto t) {
        using T = decltype(t);
        return launch_logprobs<T>(p, a, static_cast<const T*>(logits), static_cast<T*>(grad_logits), temp, stream);
    });
}

gsx_hip_status gsx_hip_log_probs_backward(const void* logits, int32_t logits_type, int64_t logits_stride, int64_t rows,
                                          int64_t vocab, const int32_t* ids, float temperature, const float* row_stats,
                                          const float* row_grad, float grad_scale, const float* entropy_grad,
                                          float entropy_scale, void* grad_logits, int64_t grad_stride, hipStream_t stream) {
    LogProbsArgs a = logprobs_args(logits_stride, rows, vocab, ids, temperature, row_grad, grad_scale, entropy_grad,
                                   entropy_scale, grad_stride);
    a.stats = const_cast<float*>(row_stats);  // read only
    const gsx_hip_status st = logprobs_check(a, logits, logits_type, temperature, grad_logits);
    if (st != GSX_HIP_SUCCESS || rows == 0) return st;
    if (row_stats == nullptr || grad_logits == nullptr)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "log probabilities backward: null pointer");
    return with_type(logits_type, [&](auto t) {
        using T = decltype(t);
        return launch_grad<T>(a, static_cast<const T*>(logits), static_cast<T*>(grad_logits), stream);
    });
}

}  // extern "C"

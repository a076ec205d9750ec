// The first launch of what reads rows of logits once: slices of a row, each with its largest
// logit, its sums and its top candidates (and, with STATS, the rank of a given token).  The
// design: token_logprobs.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged_common.h"
#include "pulsar_paged.h"

namespace pw4 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr int kList = 1024;  // a slice's candidates that are ranked at once
constexpr int kJoin = 512;   // a row's

struct SliceSums {
    float m, z, t;  // largest logit, sum e^(x-m), sum e^(x-m) (x-m); m = -inf: no logit above -inf
    int ahead;      // logits ahead of the given token's
};

struct SliceArgs {
    const void* logits;
    const int64_t* targets;  // ranks are of these tokens
    const uint8_t* passed;   // rows whose byte is not 0 are passed over; null: none
    SliceSums* sums;      // workspace [tokens, slices]
    uint64_t* top;        // workspace [tokens, slices, top_k] keys, greatest first, 0 past the last
    int64_t row_stride;
    int32_t tokens, vocab, top_k, slices, slice;  // slice: logits of one
};

__device__ __forceinline__ float lowest_if_nan(float x) { return x == x ? x : -__builtin_inff(); }

// A logit in an order of unsigned numbers: NaN as -inf, -0 as 0; 0 is below all.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, lowest_if_nan(x) + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
// Logit and index as one number: the greater comes first among the top tokens.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)ordered(x) << 32 | ~i; }

// A vector of logits at any address that logits have.
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Logits;
template <>
struct Logits<PW4_DTYPE_F16> {
    using T = uint16_t;
    static constexpr uint16_t kLowest = 0xfc00;
    static __device__ __forceinline__ float value(uint32_t word, int j) {
        return (float)as_h2(word)[j];
    }
};
template <>
struct Logits<PW4_DTYPE_BF16> {
    using T = uint16_t;
    static constexpr uint16_t kLowest = 0xff80;
    static __device__ __forceinline__ float value(uint32_t word, int j) {
        return __builtin_bit_cast(float, j ? word & 0xffff0000u : word << 16);
    }
};
template <>
struct Logits<PW4_DTYPE_F32> {
    using T = uint32_t;
    static constexpr uint32_t kLowest = 0xff800000u;
    static __device__ __forceinline__ float value(uint32_t word, int) { return __builtin_bit_cast(float, word); }
};

template <int DT>
__device__ __forceinline__ float logit_at(const void* row, int64_t i) {
    const typename Logits<DT>::T x = static_cast<const typename Logits<DT>::T*>(row)[i];
    return Logits<DT>::value(x, 0);
}

// STATS: with rank and entropy.
template <int DT, int PER, bool STATS>
__global__ __launch_bounds__(kThreads) void slice_kernel(const SliceArgs a) {
    using L = Logits<DT>;
    using T = typename L::T;
    constexpr int kVec = 16 / sizeof(T);           // logits of a 16-byte vector
    constexpr int kVecs = PER / kVec;              // vectors of a thread
    constexpr int kPerWord = 4 / sizeof(T);
    constexpr float kLog2e = 1.4426950408889634f, kInf = __builtin_inff();
    __shared__ uint32_t s_group[64];
    __shared__ float s_sum[8];
    __shared__ int s_ahead[4], s_count, s_vectors, s_vector[kList];
    __shared__ uint64_t s_list[kList];
    __shared__ uint64_t s_best[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.y;
    if (!STATS && a.passed != nullptr && a.passed[row] != 0) return;
    const T* const x = static_cast<const T*>(a.logits) + (int64_t)row * a.row_stride;
    const int begin = blockIdx.x * a.slice, end = min(begin + a.slice, a.vocab);
    // the aligned part, and the odd logits around it; or, without STATS, vectors from the slice's start on,
    // whatever its address: equal rows then have equal sums, to the bit
    const int to_aligned = STATS ? (int)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15)) % 16 / sizeof(T)) : 0;
    const int first = min(begin + to_aligned, end), vectors = (end - first) / kVec;
    const int head = first - begin, tail = first + vectors * kVec;
    const int odd_at = tid < head ? begin + tid : tail + tid - head;
    const bool has_odd = odd_at < end && (tid < head || odd_at >= tail);
    u32x4 held[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        constexpr uint32_t low = sizeof(T) == 2 ? L::kLowest * 0x10001u : (uint32_t)L::kLowest;
        held[v] = u32x4{low, low, low, low};
        if (v * kThreads + tid < vectors) {
            using Vec = std::conditional_t<STATS, u32x4, std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>>;
            held[v] = *reinterpret_cast<const Vec*>(x + first + (v * kThreads + tid) * kVec);
        }
    }
    const float odd = has_odd ? logit_at<DT>(x, odd_at) : -kInf;
    __builtin_amdgcn_sched_barrier(0);  // nothing waits for the target ahead of the loads
    const int64_t target = STATS ? a.targets[row] : -1;
    const bool given = STATS && target >= 0 && target < a.vocab;
    const float mine = given ? lowest_if_nan(logit_at<DT>(x, target)) : kInf;
    const int my_first = first + tid * kVec;  // index of vector 0's first logit
    // Logit e of vector v.  (Its words are made opaque before each use of a vector, so that a
    // later one takes them apart again, rather than have every value held in between.)
    auto logit = [&](int v, int e) { return L::value(held[v][e / kPerWord], e % kPerWord); };
    // f(logit, index) of the thread's own logits, from memory: for what is rare
    auto each_again = [&](auto&& f) {
        for (int i = my_first; i < tail; i += kThreads * kVec) {
#pragma clang loop unroll(disable)
            for (int e = 0; e < kVec; ++e) f(logit_at<DT>(x, i + e), i + e);
        }
        if (has_odd) f(odd, odd_at);
    };
    float m = lowest_if_nan(odd), peak[kVecs];  // the vectors' largest logits (NaN passed over)
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        asm volatile("" : "+v"(held[v]));
        peak[v] = -kInf;
#pragma unroll
        for (int e = 0; e < kVec; ++e) peak[v] = fmaxf(peak[v], logit(v, e));
        m = fmaxf(m, peak[v]);
    }
    // ---- the slice's largest logit, and a bound that its top_k reach
    uint32_t g = ordered(m);
    g = max(g, (uint32_t)__shfl_xor((int)g, 1));
    g = max(g, (uint32_t)__shfl_xor((int)g, 2));
    if ((tid & 3) == 0) s_group[tid >> 2] = g;
    if (tid == 0) s_count = s_vectors = 0;
    __syncthreads();
    g = s_group[lane];
    m = wave_max(unordered(g));
    uint32_t bound = 0;
    if (a.top_k > 0) {  // the greatest number of 16 bits, and then zeros, that top_k groups reach
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t higher = bound | 1u << bit;
            if (__popcll(__ballot(g >= higher)) >= a.top_k) bound = higher;
        }
    }
    const float lowest = a.top_k > 0 ? unordered(max(bound, 0x007fffffu)) : kInf;
    // ---- sums, rank, and the logits that reach the bound
    const float shift = m == -kInf ? 0.f : m;
    float z = 0.f, t = 0.f;
    int ahead = 0;
    bool tie = false;
    auto add = [&](float l) {
        // the difference first: l * log2(e) alone would round, and overflow, by the logit's size
        const float d = l - shift, e = __builtin_amdgcn_exp2f(d * kLog2e);
        z += e;
        if (STATS) t = __builtin_fmaf(e, fmaxf(d, -1e30f), t);  // 0 * -inf is no term
    };
    const bool listing = a.top_k > 0;
    auto reaching = [&](float l) { return listing && !(l < lowest); };
    auto candidate = [&](float l, int i) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kList) s_list[at] = key_of(l, (uint32_t)i);
    };
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        __builtin_amdgcn_sched_barrier(0);  // a vector at a time
        asm volatile("" : "+v"(held[v]));
#pragma unroll
        for (int e = 0; e < kVec; ++e) add(logit(v, e));
        if (STATS && __any(peak[v] >= mine)) {  // for a likely token, few vectors
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                ahead += __popcll(__ballot(logit(v, e) > mine));
                tie |= logit(v, e) == mine;
            }
        }
        if (reaching(peak[v]) && v * kThreads + tid < vectors) {
            const int at = atomicAdd(&s_vectors, 1);
            if (at < kList) s_vector[at] = my_first + v * kThreads * kVec;
        }
    }
    add(odd);
    if (STATS) {
        ahead += __popcll(__ballot(odd > mine));
        tie |= odd == mine;
    }
    if (has_odd && reaching(odd)) candidate(odd, odd_at);
    if (given && __any(tie)) {
        int before = 0;
        each_again([&](float l, int i) { before += l == mine && i < (int)target; });
        ahead += wave_sum(before);
    }
    z = wave_sum(z);
    if (STATS) t = wave_sum(t);
    if (lane == 0) {
        s_sum[wave] = z;
        s_sum[4 + wave] = t;
        s_ahead[wave] = ahead;
    }
    __syncthreads();
    const int64_t out = (int64_t)row * a.slices + blockIdx.x;
    if (tid == 0) {
        a.sums[out] = SliceSums{m, (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]),
                                (s_sum[4] + s_sum[5]) + (s_sum[6] + s_sum[7]),
                                (s_ahead[0] + s_ahead[1]) + (s_ahead[2] + s_ahead[3])};
    }
    if (a.top_k == 0) return;
    uint64_t* const top = a.top + out * a.top_k;
    // the candidates of the vectors that reach the bound, a logit a thread
    int count = s_vectors;
    if (count <= kList) {
        for (int j = tid; j < count * kVec; j += kThreads) {
            const int i = s_vector[j / kVec] + j % kVec;
            const float l = logit_at<DT>(x, i);
            if (!(l < lowest)) candidate(l, i);
        }
        __syncthreads();
        count = s_count;
    }
    if (count > kList) {
        // Ties, as masks make them.  With the bound's last bits, what is above it lies in fewer
        // than top_k groups; of what equals it the first top_k are enough.
        for (int bit = 15; bit >= 0; --bit) {
            const uint32_t higher = bound | 1u << bit;
            if (__popcll(__ballot(g >= higher)) >= a.top_k) bound = higher;
        }
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        each_again([&](float l, int i) {
            if (ordered(l) > bound) candidate(l, i);
        });
        if (wave == 0) {
            int found = 0;
            for (int i0 = begin; i0 < end && found < a.top_k; i0 += 64) {
                const int i = i0 + lane;
                const float l = i < end ? logit_at<DT>(x, i) : 0.f;
                const bool equal = i < end && ordered(l) == bound;
                const uint64_t all = __ballot(equal);
                if (equal && found + __popcll(all & ((1ull << lane) - 1)) < a.top_k) candidate(l, i);
                found += __popcll(all);
            }
        }
        __syncthreads();
        count = s_count;
    }
    if (count <= kList) {
        for (int i = tid; i < max(count, a.top_k); i += kThreads) {
            if (i >= count) {
                top[i] = 0;
                continue;
            }
            const uint64_t key = s_list[i];
            int place = 0;
            for (int j = 0; j < count; ++j) place += s_list[j] > key;
            if (place < a.top_k) top[place] = key;
        }
        return;
    }
    uint64_t below = ~0ull;  // more above the bound than the list holds: one token a round
    for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
        each_again([&](float l, int i) {
            const uint64_t key = key_of(l, (uint32_t)i);
            if (key < below && key > best) best = key;
        });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, d);
            best = other > best ? other : best;
        }
        if (lane == 0) s_best[wave] = best;
        __syncthreads();
        below = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
        if (tid == 0) top[k] = below;
        __syncthreads();
    }
}

// A row's top_k keys from its slices', `tops` [slices, top_k]: store(place, key), by one wave.  `mine`
// is JOIN keys of the wave's in LDS.
template <int JOIN = kJoin, typename F>
__device__ __forceinline__ void join_tops(const uint64_t* tops, int slices, int top_k, uint64_t* mine, F&& store) {
    const int lane = threadIdx.x & 63, keys = slices * top_k;
    // A number that the q-th greatest keys of at least top_k / q slices reach is a bound for the
    // row, which top_k keys at least reach: the few that do are ranked.  (q is 1 where there are
    // top_k slices; a lane's number is the greatest of the slices that it has.)
    const int q = (top_k + slices - 1) / slices, reach = (top_k + q - 1) / q;
    uint32_t bound = 0, g = 0;
    for (int s = lane; s < slices; s += 64) g = max(g, (uint32_t)(tops[(int64_t)s * top_k + q - 1] >> 32));
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t higher = bound | 1u << bit;
        if (__popcll(__ballot(g >= higher)) >= reach) bound = higher;
    }
    int count = 0;
    for (int i0 = 0; i0 < keys; i0 += 64) {
        const uint64_t key = i0 + lane < keys ? tops[i0 + lane] : 0;
        const bool reaches = key != 0 && (uint32_t)(key >> 32) >= bound;
        const uint64_t all = __ballot(reaches);
        const int at = count + __popcll(all & ((1ull << lane) - 1));
        if (reaches && at < JOIN) mine[at] = key;
        count += __popcll(all);
    }
    if (count <= JOIN) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < count; i += 64) {
            const uint64_t key = mine[i];
            int place = 0;
            for (int j = 0; j < count; ++j) place += mine[j] > key;
            if (place < top_k) store(place, key);
        }
        return;
    }
    uint64_t below = ~0ull;  // many keys that tie at the bound: one token a round
    for (int k = 0; k < top_k; ++k) {
        uint64_t best = 0;
        for (int i = lane; i < keys; i += 64) {
            const uint64_t key = tops[i];
            if (key < below && key > best) best = key;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, d);
            best = other > best ? other : best;
        }
        below = best;
        if (lane == 0) store(k, best);
    }
}

// Logits of a thread: 32, or 16 where slices of 32 leave half of the CUs without one.
inline int per_thread(int64_t tokens, int64_t vocab) {
    return 2 * tokens * ceil_div(vocab, kThreads * 32) <= device_cus() ? 16 : 32;
}
// Slices of one size; the odd logits come on top of the vectors.
inline int slices_of(int64_t tokens, int64_t vocab) { return (int)ceil_div(vocab, kThreads * per_thread(tokens, vocab)); }

inline size_t sums_bytes(int64_t tokens, int64_t slices) { return (size_t)round_up(tokens * slices * (int64_t)sizeof(SliceSums), 16); }

}  // namespace
}  // namespace pw4

// New keys and values on their way into a paged cache: rotated by their positions, and
// rounded to the cache's 16 bits or to its blocks of 4; and what a 4-bit cache holds, read
// back.  (The formulas and the pages' layout: pulsar_paged.h.)
//
// A thread has sixteen elements of a head, eight and the eight that they are paired with, at a
// number of the token's heads in turn, with the pairs' cosines and sines in registers; the next
// head's elements are under way meanwhile.  What vectors of eight do not fit (odd rotations, odd
// addresses) is done one element at a time by append_any_kernel: 16384 tokens, 32 heads on 8 of 80, of which 20 or
// 40 elements rotate, take 131 us (1.9 TB/s), and 56 (4.6) where all 80 do.
//
// Rotations are fp64: the product of an element and an fp32 cosine is exact there, so the sum is
// rounded once and a 4-bit cache's exponent and codes, which stand next to borders, do not depend
// on the order of the operations.  fp64 vector instructions run at fp32's rate on this chip.
//
// A block of 32 elements is four vectors of two to four threads of a wave; its largest magnitude
// takes one or two exchanges.  The conversion instruction rounds to codes by the block's scale (to
// nearest, halves to even, saturating), two elements each.
//
// Bound by memory: 232 MB in and out (8 chunks of up to 2048 tokens, 32 heads of 128 and twice 8, 16
// bits) take 53 us, 4.4 TB/s where a copy reaches 4.9; vector units are busy 33% of the cycles, into
// 4 bits 41%.  A thread's several heads share what depends on the token and the lane (place, angles,
// neighbours): with a head a thread a prompt into 4 bits took 131 us, with several 85, chunks into 16
// bits 66 and 53.  A few tokens are bound by the launch and two loads in turn: 64 tokens take 3.8 us under a
// profiler, 7.8 a call.
#include "pulsar_paged.h"

#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged_common.h"

using namespace pw4;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMostGroups = 1 << 22;  // of a launch: threads are counted in 32 bits, and past 2^32 tokens are lost

struct Heads {
    const uint16_t* from;
    int64_t token, head;  // strides, elements
};
struct AppendArgs {
    Heads q, k, v;
    uint16_t* q_out;
    uint8_t* k_cache;
    uint8_t* v_cache;
    const int64_t* slots;
    const int64_t* positions;
    const float* rope;
    int64_t page_bytes, row_bytes, head_bytes;         // 16-bit caches
    uint32_t row_codes, row_exps, exps_at;             // 4-bit caches
    int64_t places;                                    // slots of the pool
    int64_t rope_rows;
    int32_t q_heads, kv_heads, dim, rot, page_size, interleaved;
    int32_t exp_limit;                                 // greatest exponent byte
    int32_t tokens, abreast;                           // append_kernel: head groups of a token side by side
};

template <bool BF16>
__device__ __forceinline__ float widen16(uint16_t u) {
    if constexpr (BF16) {
        return __builtin_bit_cast(float, (uint32_t)u << 16);
    } else {
        return (float)__builtin_bit_cast(_Float16, u);
    }
}

// The largest magnitude among fp32 elements, as its bits (a NaN or an infinity: 0x7f800000 or more).
__device__ __forceinline__ uint32_t magnitude(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    return top;
}
// The exponent byte of a block whose largest magnitude is `top`: that magnitude's exponent, one more from
// 1.75 of it on, less 2.
__device__ __forceinline__ uint32_t exponent_of(uint32_t top, int limit) {
    return top >= 0x7f800000u ? 255u : (uint32_t)min(max((int)((top + 0x200000u) >> 23) - 2, 0), limit);
}
__device__ __forceinline__ uint32_t to_codes(const float (&x)[8], uint32_t exp) {
    const float scale = __builtin_bit_cast(float, exp << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    return w;
}
__device__ __forceinline__ uint32_t other_lane(uint32_t v, int lane) { return (uint32_t)__shfl((int)v, lane); }

// Where a token goes.
struct Token {
    bool known, stored;       // its position is in the table; and its slot in the pool
    const float* table;       // its cosines and sines
    uint32_t page, row;
};
__device__ __forceinline__ Token token_at(const AppendArgs& a, int token) {
    Token t{true, false, nullptr, 0, 0};
    const int64_t slot = a.slots[token];
    t.stored = slot >= 0 && slot < a.places;
    if (a.positions != nullptr) {
        const int64_t p = a.positions[token];
        t.known = p >= 0 && p < a.rope_rows;
        if (t.known) t.table = a.rope + p * a.rot;
        t.stored &= t.known;
    }
    if (t.stored) {
        t.page = (uint32_t)slot / (uint32_t)a.page_size;
        t.row = (uint32_t)slot - t.page * (uint32_t)a.page_size;
    }
    return t;
}
// Head h of a token's: q's first, then k's, then v's.
struct Head {
    bool is_q, is_v;
    int at;
    const uint16_t* from;
    __device__ __forceinline__ Head(const AppendArgs& a, int token, int h) {
        is_q = h < a.q_heads;
        is_v = h >= a.q_heads + a.kv_heads;
        at = is_q ? h : is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
        const Heads& heads = is_q ? a.q : is_v ? a.v : a.k;
        from = heads.from + token * heads.token + at * heads.head;
    }
};

template <bool BF16>
__device__ __forceinline__ void widen8(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = widen16<BF16>((uint16_t)(w[e / 2] >> (e % 2 * 16)));
}
template <bool BF16>
__device__ __forceinline__ u32x4 round8(const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = f32_to_out<BF16>(x[2 * e]) | (uint32_t)f32_to_out<BF16>(x[2 * e + 1]) << 16;
    return w;
}

// Everything 16-byte aligned, head_dim and rot multiples of 16.  A wave is 64 / U rows of U = dim / 16
// lanes; a row of lanes goes over heads first, first + abreast, ... of its token, its lane u having
// elements 8 u .. + 7 and their mates rot / 2 further on, or (PAIRS, values, and what is not rotated)
// 16 u .. + 15.
template <bool BF16, bool FP4, bool PAIRS>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 63, units = a.dim / 16, in_wave = 64 / units;
    const int r = lane / units, u = lane - r * units, row0 = lane - u;
    const int group = ((int)threadIdx.x >> 6) * in_wave + r, side = group / a.abreast;
    const int at_once = kThreads / 64 * in_wave / a.abreast;  // tokens
    const int token = (int)blockIdx.x * at_once + side;
    if (r >= in_wave || side >= at_once || token >= a.tokens) return;
    const int heads = a.q_heads + 2 * a.kv_heads, step = a.abreast * (int)gridDim.y;
    int h = group - side * a.abreast + (int)blockIdx.y * a.abreast;
    if (h >= heads) return;
    const int half = a.rot / 2;
    const bool turns = a.positions != nullptr && 16 * u < a.rot, split = !PAIRS && turns;
    const int d0 = split ? 8 * u : 16 * u, d1 = split ? half + 8 * u : 16 * u + 8;
    const auto load = [&](int head, u32x4 (&w)[2]) {
        const Head x(a, token, head);
        w[0] = *reinterpret_cast<const u32x4*>(x.from + (x.is_v ? 16 * u : d0));
        w[1] = *reinterpret_cast<const u32x4*>(x.from + (x.is_v ? 16 * u + 8 : d1));
    };
    u32x4 next[2];
    load(h, next);
    const Token t = token_at(a, token);
    double c[8], s[8];
    if (turns && t.known) {
        float cf[8], sf[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<f32x4*>(cf + e) = *reinterpret_cast<const f32x4*>(t.table + 8 * u + e);
            *reinterpret_cast<f32x4*>(sf + e) = *reinterpret_cast<const f32x4*>(t.table + half + 8 * u + e);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            c[e] = cf[e];
            s[e] = sf[e];
        }
    }
    // the lanes and halves that hold the neighbours of the lane's two vectors in a block of 32
    int near0[2], near1[2];      // by 8 elements and by 16: lane
    bool late0[2], late1[2];     // whether it is that lane's second vector
    if (FP4 && !PAIRS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const auto owner = [&](int d, int& where, bool& late) {
                const bool turned = a.positions != nullptr && d < a.rot;
                late = turned ? d >= half : d % 16 != 0;
                where = row0 + (turned ? (d - (late ? half : 0)) / 8 : d / 16);
            };
            owner(d0 ^ (8 << i), near0[i], late0[i]);
            owner(d1 ^ (8 << i), near1[i], late1[i]);
        }
    }
    while (true) {
        const u32x4 w[2] = {next[0], next[1]};
        const Head x(a, token, h);
        const bool more = h + step < heads;
        if (more) load(h + step, next);
        const bool turned = turns && t.known && !x.is_v;
        float x0[8], x1[8];
        if (turned || (FP4 && !x.is_q)) {
            widen8<BF16>(w[0], x0);
            widen8<BF16>(w[1], x1);
        }
        if (turned) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float& fa = PAIRS ? (e < 4 ? x0 : x1)[e % 4 * 2] : x0[e];
                float& fb = PAIRS ? (e < 4 ? x0 : x1)[e % 4 * 2 + 1] : x1[e];
                const double da = fa, db = fb;
                fa = (float)__builtin_fma(da, c[e], -(db * s[e]));
                fb = (float)__builtin_fma(db, c[e], da * s[e]);
            }
        }
        if (x.is_q || (!FP4 && t.stored)) {
            u32x4 out0 = w[0], out1 = w[1];
            if (turned) {
                out0 = round8<BF16>(x0);
                out1 = round8<BF16>(x1);
            } else if (!t.known) {
                out0 = out1 = u32x4{0, 0, 0, 0};
            }
            const int64_t in_cache = t.page * a.page_bytes + t.row * a.row_bytes + x.at * a.head_bytes;
            uint16_t* const to = x.is_q ? a.q_out + ((int64_t)token * a.q_heads + x.at) * a.dim
                                        : reinterpret_cast<uint16_t*>((x.is_v ? a.v_cache : a.k_cache) + in_cache);
            *reinterpret_cast<u32x4*>(to + (x.is_v ? 16 * u : d0)) = out0;
            *reinterpret_cast<u32x4*>(to + (x.is_v ? 16 * u + 8 : d1)) = out1;
        } else if (FP4 && t.stored) {
            uint32_t m0 = magnitude(x0), m1 = magnitude(x1);
            if (PAIRS || x.is_v || a.positions == nullptr) {  // (a row's lanes agree)
                m0 = max(m0, m1);
                m0 = m1 = max(m0, other_lane(m0, lane ^ 1));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t a0 = other_lane(m0, near0[i]), a1 = other_lane(m1, near0[i]);
                    const uint32_t b0 = other_lane(m0, near1[i]), b1 = other_lane(m1, near1[i]);
                    m0 = max(m0, late0[i] ? a1 : a0);
                    m1 = max(m1, late1[i] ? b1 : b0);
                }
            }
            const int at0 = x.is_v ? 16 * u : d0, at1 = x.is_v ? 16 * u + 8 : d1;
            const uint32_t e0 = exponent_of(m0, a.exp_limit), e1 = exponent_of(m1, a.exp_limit);
            uint8_t* const to = (x.is_v ? a.v_cache : a.k_cache) + t.page * a.page_bytes;
            const uint32_t place = x.at * a.page_size + t.row;
            uint8_t* const codes = to + place * a.row_codes;
            uint8_t* const exps = to + a.exps_at + place * a.row_exps;
            *reinterpret_cast<uint32_t*>(codes + at0 / 2) = to_codes(x0, e0);
            *reinterpret_cast<uint32_t*>(codes + at1 / 2) = to_codes(x1, e1);
            if (at0 % 32 == 0) exps[at0 / 32] = (uint8_t)e0;
            if (at1 % 32 == 0) exps[at1 / 32] = (uint8_t)e1;
        }
        if (!more) return;
        h += step;
    }
}

// ---- one element at a time -------------------------------------------------------

// What eight neighbouring elements, from element d0 of a head on, are rotated by: element e becomes
// own * c[e] + mate * s[e], its mate being element mate(e) of the head.
struct Turn {
    float c[8], s[8];
    int d0, rot, half;
    bool any, pairs;

    __device__ __forceinline__ Turn(const AppendArgs& a, const float* table, int d0_) : d0(d0_), rot(a.rot), half(a.rot / 2) {
        any = table != nullptr && d0 < rot;
        pairs = a.interleaved;
        if (!any) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = min(d0 + e, rot - 1), i = pairs ? d / 2 : d < half ? d : d - half;
            const bool first = pairs ? d % 2 == 0 : d < half;
            c[e] = table[i];
            s[e] = first ? -table[half + i] : table[half + i];
        }
    }
    __device__ __forceinline__ int mate(int e) const {
        const int d = d0 + e;
        if (d >= rot) return d;
        return pairs ? d ^ 1 : d < half ? d + half : d - half;
    }
    // The rotated elements of a head, rounded to fp32.
    template <bool BF16>
    __device__ __forceinline__ void apply(const uint16_t* head, float (&x)[8]) const {
        float other[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) other[e] = widen16<BF16>(head[mate(e)]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double turned = __builtin_fma((double)x[e], (double)c[e], (double)other[e] * (double)s[e]);
            x[e] = d0 + e < rot ? (float)turned : x[e];
        }
    }
};

// Tokens blockIdx.x, + gridDim.x, ...; of their heads blockIdx.y's share.  A thread has eight neighbouring
// elements of a head; four threads have a block of 32.
template <bool BF16, bool FP4>
__device__ __forceinline__ void append_token(const AppendArgs& a, int token) {
    const int units = a.dim / 8, at_once = kThreads / units;
    const int first = threadIdx.x / units, d0 = (threadIdx.x - first * units) * 8;
    if (first >= at_once) return;
    const Token t = token_at(a, token);
    const Turn turn(a, t.table, d0);
    const int heads = a.q_heads + 2 * a.kv_heads;
    for (int h = first + blockIdx.y * at_once; h < heads; h += at_once * gridDim.y) {
        const Head x(a, token, h);
        if (!x.is_q && !t.stored) continue;
        uint16_t own[8];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) own[e] = x.from[d0 + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = widen16<BF16>(own[e]);
        const bool turns = turn.any && !x.is_v;
        if (turns) turn.template apply<BF16>(x.from, f);
        if (FP4 && !x.is_q) {
            uint32_t top = magnitude(f);
            top = max(top, other_lane(top, (threadIdx.x & 63) ^ 1));
            top = max(top, other_lane(top, (threadIdx.x & 63) ^ 2));
            const uint32_t exp = exponent_of(top, a.exp_limit);
            uint8_t* const to = (x.is_v ? a.v_cache : a.k_cache) + t.page * a.page_bytes;
            const uint32_t place = x.at * a.page_size + t.row;
            *reinterpret_cast<uint32_t*>(to + place * a.row_codes + d0 / 2) = to_codes(f, exp);
            if (d0 % 32 == 0) to[a.exps_at + place * a.row_exps + d0 / 32] = (uint8_t)exp;
            continue;
        }
        uint16_t* to = a.q_out + ((int64_t)token * a.q_heads + x.at) * a.dim;
        if (!x.is_q) {
            to = reinterpret_cast<uint16_t*>((x.is_v ? a.v_cache : a.k_cache) + t.page * a.page_bytes + t.row * a.row_bytes +
                                             x.at * a.head_bytes);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) to[d0 + e] = !t.known ? 0 : turns ? f32_to_out<BF16>(f[e]) : own[e];
    }
}
template <bool BF16, bool FP4>
__global__ __launch_bounds__(kThreads) void append_any_kernel(const AppendArgs a) {
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) append_token<BF16, FP4>(a, (int)token);
}

struct ReadArgs {
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const int64_t* slots;
    uint16_t* k;
    uint16_t* v;
    int64_t page_bytes, places;
    uint32_t row_codes, row_exps, exps_at;
    int32_t kv_heads, dim, page_size, tokens;
};

// A token's keys' and values' words of eight codes.  (16384 tokens of twice 8 heads of 96, 64 MB in
// and out, 18.5 us, 3.5 TB/s; waves waiting for memory 63% of their time.)
template <bool BF16>
__device__ __forceinline__ void read_token(const ReadArgs& a, int token) {
    const int units = a.dim / 8, items = 2 * a.kv_heads * units;
    const int64_t slot = a.slots[token];
    const bool there = slot >= 0 && slot < a.places;
    const uint32_t page = there ? (uint32_t)slot / (uint32_t)a.page_size : 0;
    const uint32_t row = there ? (uint32_t)slot - page * (uint32_t)a.page_size : 0;
    for (int i = threadIdx.x + blockIdx.y * kThreads; i < items; i += kThreads * gridDim.y) {
        const int h = i / units, d0 = (i - h * units) * 8;
        const bool is_v = h >= a.kv_heads;
        const int at = is_v ? h - a.kv_heads : h;
        u32x4 out{0, 0, 0, 0};
        if (there) {
            const uint8_t* const from = (is_v ? a.v_cache : a.k_cache) + page * a.page_bytes;
            const uint32_t place = at * a.page_size + row;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(from + place * a.row_codes + d0 / 2);
            const float scale = __builtin_bit_cast(float, (uint32_t)from[a.exps_at + place * a.row_exps + d0 / 32] << 23);
            if constexpr (BF16) {
                out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
                out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
                out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
                out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
            } else {
                out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
                out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
                out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
                out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
            }
        }
        *reinterpret_cast<u32x4*>((is_v ? a.v : a.k) + ((int64_t)token * a.kv_heads + at) * a.dim + d0) = out;
    }
}
template <bool BF16>
__global__ __launch_bounds__(kThreads) void read_kernel(const ReadArgs a) {
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) read_token<BF16>(a, (int)token);
}

// ---- host ----------------------------------------------------------------------

bool small(int64_t v) { return v >= 0 && v <= INT_MAX; }

// A page of a 4-bit cache: sizes that 32 bits hold.
int check_fp4_pages(const void* k_cache, const void* v_cache, int64_t kv_heads, int64_t dim, int64_t pages, int64_t page_size,
                    int64_t page_stride) {
    if (dim % 32 != 0 || !small(kv_heads) || page_size > INT_MAX / 256 / std::max<int64_t>(kv_heads, 1)) return PW4_ERR_SHAPE;
    if ((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) != 0 || page_stride < 0 || page_stride % 16 != 0) return PW4_ERR_ARG;
    if (page_stride > INT_MAX || (pages > 1 && page_stride < page_size * kv_heads * (dim / 2 + dim / 32))) return PW4_ERR_SHAPE;
    return PW4_OK;
}

int append(const pw4_paged_append_args* a, bool fp4, pw4_stream_t stream) {
    if (a == nullptr || (a->dtype != PW4_DTYPE_F16 && a->dtype != PW4_DTYPE_BF16)) return PW4_ERR_ARG;
    if (a->num_tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->head_dim <= 0 || a->num_pages < 0 || a->page_size <= 0 ||
        a->rope_rows < 0 || a->rot < 0) {
        return PW4_ERR_ARG;
    }
    if (!small(a->num_tokens) || a->head_dim % 8 != 0 || a->head_dim > 256 || a->rot % 2 != 0 || a->rot > a->head_dim ||
        !small(a->page_size) || !small(a->num_pages) || !small(a->num_pages * a->page_size) || !small(a->rope_rows) ||
        a->q_heads > 65535 || a->kv_heads > 65535) {
        return PW4_ERR_SHAPE;
    }
    if (fp4) {
        if (const int rc = check_fp4_pages(a->k_cache, a->v_cache, a->kv_heads, a->head_dim, a->num_pages, a->page_size, a->page_stride)) {
            return rc;
        }
    }
    const bool q = a->q != nullptr, turns = a->positions != nullptr;
    const int64_t heads = (q ? a->q_heads : 0) + 2 * a->kv_heads;
    if (a->num_tokens == 0 || heads == 0) return PW4_OK;
    if (!a->slots || (a->kv_heads && (!a->k || !a->v || (a->num_pages && (!a->k_cache || !a->v_cache))))) return PW4_ERR_ARG;
    if (turns ? !a->rope && a->rope_rows * a->rot != 0 : a->rope != nullptr || q) return PW4_ERR_ARG;
    if (q && (!a->q_out || (uintptr_t)a->q_out % 16 != 0)) return PW4_ERR_ARG;
    if ((uintptr_t)a->rope % 4 != 0) return PW4_ERR_ARG;
    const uint64_t caches = fp4 ? 0 : (uint64_t)(uintptr_t)a->k_cache | (uint64_t)(uintptr_t)a->v_cache;
    const uint64_t cache_strides = fp4 ? 0 : (uint64_t)(a->page_stride | a->row_stride | a->kv_head_stride);
    const uint64_t addresses = (q ? (uint64_t)(uintptr_t)a->q : 0) | (uint64_t)(uintptr_t)a->k | (uint64_t)(uintptr_t)a->v | caches;
    const uint64_t strides = (q ? (uint64_t)(a->q_token_stride | a->q_head_stride) : 0) |
                             (uint64_t)(a->k_token_stride | a->k_head_stride | a->v_token_stride | a->v_head_stride) | cache_strides;
    if (addresses & 1) return PW4_ERR_ARG;
    // vectors of eight: everything aligned, and whole vectors rotated or not
    const bool vec = (addresses & 15) == 0 && (strides & 7) == 0 && a->head_dim % 16 == 0 &&
                     (!turns || (a->rot % 16 == 0 && (uintptr_t)a->rope % 16 == 0));
    AppendArgs p{};
    p.q = Heads{static_cast<const uint16_t*>(a->q), a->q_token_stride, a->q_head_stride};
    p.k = Heads{static_cast<const uint16_t*>(a->k), a->k_token_stride, a->k_head_stride};
    p.v = Heads{static_cast<const uint16_t*>(a->v), a->v_token_stride, a->v_head_stride};
    p.q_out = static_cast<uint16_t*>(a->q_out);
    p.k_cache = static_cast<uint8_t*>(a->k_cache);
    p.v_cache = static_cast<uint8_t*>(a->v_cache);
    p.slots = a->slots;
    p.positions = a->positions;
    p.rope = a->rope;
    p.page_bytes = fp4 ? a->page_stride : a->page_stride * 2;
    p.row_bytes = a->row_stride * 2;
    p.head_bytes = a->kv_head_stride * 2;
    p.row_codes = (uint32_t)a->head_dim / 2;
    p.row_exps = (uint32_t)a->head_dim / 32;
    p.exps_at = (uint32_t)(a->kv_heads * a->page_size * (a->head_dim / 2));
    p.places = a->num_pages * a->page_size;
    p.rope_rows = a->rope_rows;
    p.q_heads = q ? (int32_t)a->q_heads : 0;
    p.kv_heads = (int32_t)a->kv_heads;
    p.dim = (int32_t)a->head_dim;
    p.rot = (int32_t)a->rot;
    p.page_size = (int32_t)a->page_size;
    p.interleaved = a->interleaved != 0;
    p.exp_limit = a->dtype == PW4_DTYPE_F16 ? 127 + 13 : 127 + 125;  // 6 * 2^e is finite in the type, 4 * 2^(e + 1) is not
    p.tokens = (int32_t)a->num_tokens;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const auto run = [&](auto bf16, auto four) {
        constexpr bool BF16 = decltype(bf16)::value, FP4 = decltype(four)::value;
        if (!vec) {
            const int64_t passes = ceil_div(heads, kThreads / (a->head_dim / 8));
            // Several workgroups a token and one, us, heads of 80, 20 elements rotated: 1 token 3.6 and 4.3, 64 3.9 and
            // 4.6, 256 4.9 and 4.9, 512 7.4 and 7.0, 1024 (the last one shared) 12.4 and 10.0, 2048 22 and 17.
            const int64_t shares = a->num_tokens * passes <= 8 * device_cus() ? passes : 1;
            hipLaunchKernelGGL((append_any_kernel<BF16, FP4>), dim3((unsigned)std::min(a->num_tokens, kMostGroups), (unsigned)shares),
                               dim3(kThreads), 0, s, p);
            return;
        }
        // Rows of lanes of a workgroup, and how many of them share a token: all, each with a head, where
        // tokens are few; else 8, so that a row's cosines serve several heads.  A head a row and 8 rows a token, us,
        // 32 heads on 8 (the rule goes over between the last two of each): heads of 128, 64 tokens 3.0 and 6.2, 512
        // 5.8 and 8.6, 1024 9.1 and 9.3, 2048 13.6 and 11.7, into 4 bits 3.6 and 6.8, 6.4 and 9.0, 10.5 and 9.8, 16.6
        // and 12.0; of 256, 512 tokens 8.9 and 9.3, 1024 13.2 and 12.1.  16384 tokens by 2, 4, 8, 16 and 32 rows a
        // token: heads of 128 92, 87, 83, 79 and 85, into 4 bits 80, 76, 75, 78 and 99; of 96 75, 72, 64, 68 and 80;
        // of 256, 16 on 4, 88, 83, 80, 85 and 85; of 64, 14 on 2, 22, 19, 21, 24 and 23.
        const int64_t rows = kThreads / 64 * (64 / (a->head_dim / 16));
        const bool few = a->num_tokens * heads <= 8 * device_cus() * rows;
        p.abreast = (int32_t)std::min<int64_t>(few ? rows : std::min<int64_t>(8, rows), heads);
        const int64_t at_once = rows / p.abreast, most = kMostGroups * at_once;  // tokens of a workgroup, of a launch
        for (int64_t first = 0; first < a->num_tokens; first += most) {
            AppendArgs part = p;
            part.tokens = (int32_t)std::min(most, a->num_tokens - first);
            part.slots += first;
            if (turns) part.positions += first;
            part.k.from += first * part.k.token;
            part.v.from += first * part.v.token;
            if (q) {
                part.q.from += first * part.q.token;
                part.q_out += first * a->q_heads * a->head_dim;
            }
            const dim3 grid((unsigned)ceil_div(part.tokens, at_once), (unsigned)(few ? ceil_div(heads, p.abreast) : 1));
            if (p.interleaved || !turns) {
                hipLaunchKernelGGL((append_kernel<BF16, FP4, true>), grid, dim3(kThreads), 0, s, part);
            } else {
                hipLaunchKernelGGL((append_kernel<BF16, FP4, false>), grid, dim3(kThreads), 0, s, part);
            }
        }
    };
    const auto with_bits = [&](auto bf16) { fp4 ? run(bf16, std::true_type{}) : run(bf16, std::false_type{}); };
    a->dtype == PW4_DTYPE_BF16 ? with_bits(std::true_type{}) : with_bits(std::false_type{});
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // namespace

extern "C" {

int pw4_paged_cache_append(const pw4_paged_append_args* args, pw4_stream_t stream) { return append(args, false, stream); }

int pw4_paged_cache_append_fp4(const pw4_paged_append_args* args, pw4_stream_t stream) { return append(args, true, stream); }

int pw4_paged_cache_read_fp4(const void* k_cache, const void* v_cache, const int64_t* slots, void* k, void* v,
                             int64_t num_tokens, int64_t kv_heads, int64_t head_dim, int64_t num_pages,
                             int64_t page_size, int64_t page_stride, int dtype, pw4_stream_t stream) {
    if (dtype != PW4_DTYPE_F16 && dtype != PW4_DTYPE_BF16) return PW4_ERR_ARG;
    if (num_tokens < 0 || kv_heads < 0 || head_dim <= 0 || num_pages < 0 || page_size <= 0) return PW4_ERR_ARG;
    if (!small(num_tokens) || head_dim > 256 || kv_heads > 65535 || !small(page_size) || !small(num_pages) ||
        !small(num_pages * page_size)) {
        return PW4_ERR_SHAPE;
    }
    if (const int rc = check_fp4_pages(k_cache, v_cache, kv_heads, head_dim, num_pages, page_size, page_stride)) return rc;
    if (num_tokens == 0 || kv_heads == 0) return PW4_OK;
    if (!slots || !k || !v || (num_pages && (!k_cache || !v_cache))) return PW4_ERR_ARG;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) != 0) return PW4_ERR_ARG;
    const ReadArgs a{static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), slots,
                     static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), page_stride, num_pages * page_size,
                     (uint32_t)head_dim / 2, (uint32_t)head_dim / 32, (uint32_t)(kv_heads * page_size * (head_dim / 2)),
                     (int32_t)kv_heads, (int32_t)head_dim, (int32_t)page_size, (int32_t)num_tokens};
    const int64_t passes = ceil_div(2 * kv_heads * (head_dim / 8), kThreads);
    // Several workgroups a token and one, us, 8 heads of 256: 1 token 2.06 and 2.18, 64 2.22 and 2.49, 256 2.48 and
    // 2.69, 512 3.1 and 3.1, 4096 10.8 and 9.3; of 128, 1 token 1.92 and 2.01, 256 2.24 and 2.36.
    const int64_t shares = num_tokens * passes <= 8 * device_cus() ? passes : 1;
    const dim3 grid((unsigned)std::min(num_tokens, kMostGroups), (unsigned)shares);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == PW4_DTYPE_BF16) {
        hipLaunchKernelGGL(read_kernel<true>, grid, dim3(kThreads), 0, s, a);
    } else {
        hipLaunchKernelGGL(read_kernel<false>, grid, dim3(kThreads), 0, s, a);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // extern "C"

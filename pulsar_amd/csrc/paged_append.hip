// New keys and values on their way into a paged cache: rotated by their positions, and
// rounded to the cache's 16 bits or to its blocks of 4; and what a 4-bit cache holds, read
// back.  (The formulas and the pages' layout: pulsar_paged.h.)
//
// A workgroup has a token, a thread eight neighbouring elements of a head at a time: it loads
// them and, of a rotated head, the eight that they are paired with (a cache line that other
// threads of the wave load as well), and goes over the token's heads with its cosines and sines
// in registers.  Pages and rows of the cache are a token's own, so their division is scalar.
//
// Rotations are fp64: the product of an element and an fp32 cosine is exact there, so the sum is
// rounded once and a 4-bit cache's exponent and codes, which stand next to borders, do not depend
// on the order of the operations.  fp64 vector instructions run at fp32's rate on this chip.
//
// Four threads hold a block of 32 elements; its largest magnitude takes two exchanges.  The
// conversion instruction rounds to codes by the block's scale (to nearest, halves to even,
// saturating), two elements each.
#include "pulsar_paged.h"

#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged_common.h"

using namespace pw4;

namespace {

constexpr int kThreads = 256;

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
};

template <bool BF16>
__device__ __forceinline__ float widen16(uint16_t u) {
    if constexpr (BF16) {
        return __builtin_bit_cast(float, (uint32_t)u << 16);
    } else {
        return (float)__builtin_bit_cast(_Float16, u);
    }
}

// Eight elements from `from` on.  VEC: it is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* from, uint16_t (&x)[8]) {
    if constexpr (VEC) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (uint16_t)(w[e / 2] >> (e % 2 * 16));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = from[e];
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* to, const uint16_t (&x)[8]) {
    if constexpr (VEC) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = x[2 * e] | (uint32_t)x[2 * e + 1] << 16;
        *reinterpret_cast<u32x4*>(to) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = x[e];
    }
}

// What a thread's eight elements, from element d0 of a head on, are rotated by: element e becomes
// own * c[e] + mate * s[e], its mate being element mate(e) of the head.
template <bool VEC>
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
    // The rotated elements of a head, rounded to fp32.  VEC: the mates of eight lie side by side,
    // and so do their cosines.
    template <bool BF16>
    __device__ __forceinline__ void apply(const uint16_t* head, const uint16_t (&own)[8], float (&out)[8]) const {
        uint16_t other[8];
        if (VEC && !pairs) {
            load8<true>(head + mate(0), other);
        } else if (VEC) {
#pragma unroll
            for (int e = 0; e < 8; ++e) other[e] = own[e ^ 1];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) other[e] = head[mate(e)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = widen16<BF16>(own[e]);
            const double turned = __builtin_fma((double)x, (double)c[e], (double)widen16<BF16>(other[e]) * (double)s[e]);
            out[e] = VEC || d0 + e < rot ? (float)turned : x;
        }
    }
};

// Eight fp32 elements of a block that this thread and the three beside it hold, to codes; the block's
// exponent byte goes to the first of the four's `exp`.
__device__ __forceinline__ uint32_t to_codes(const float (&x)[8], int limit, uint32_t& exp) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    // the exponent of the largest magnitude, one more from 1.75 of it on, less 2
    exp = top >= 0x7f800000u ? 255u : (uint32_t)min(max((int)((top + 0x200000u) >> 23) - 2, 0), limit);
    const float scale = __builtin_bit_cast(float, exp << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    return w;
}

// Token blockIdx.x; of its heads (q's, k's, v's) blockIdx.y's share.
template <bool BF16, bool VEC, bool FP4>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs a) {
    const int token = blockIdx.x;
    const int units = a.dim / 8, at_once = kThreads / units;
    const int first = threadIdx.x / units, d0 = (threadIdx.x - first * units) * 8;
    if (first >= at_once) return;
    const int64_t slot = a.slots[token];
    bool stored = slot >= 0 && slot < a.places, known = true;
    const float* table = nullptr;
    if (a.positions != nullptr) {
        const int64_t p = a.positions[token];
        known = p >= 0 && p < a.rope_rows;
        if (known) table = a.rope + p * a.rot;
        stored &= known;
    }
    const uint32_t page = stored ? (uint32_t)slot / (uint32_t)a.page_size : 0;
    const uint32_t row = stored ? (uint32_t)slot - page * (uint32_t)a.page_size : 0;
    const Turn<VEC> turn(a, table, d0);
    const int heads = a.q_heads + 2 * a.kv_heads;
    for (int h = first + blockIdx.y * at_once; h < heads; h += at_once * gridDim.y) {
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        if (!is_q && !stored) continue;
        const int at = is_q ? h : is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
        const Heads& from = is_q ? a.q : is_v ? a.v : a.k;
        const uint16_t* const head = from.from + token * from.token + at * from.head;
        uint16_t own[8];
        float x[8];
        load8<VEC>(head + d0, own);
        const bool turns = turn.any && !is_v;
        if (turns) {
            turn.template apply<BF16>(head, own, x);
        } else if (FP4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = widen16<BF16>(own[e]);
        }
        if (FP4 && !is_q) {
            uint32_t exp;
            const uint32_t codes = to_codes(x, a.exp_limit, exp);
            uint8_t* const to = (is_v ? a.v_cache : a.k_cache) + page * a.page_bytes;
            const uint32_t place = at * a.page_size + row;
            *reinterpret_cast<uint32_t*>(to + place * a.row_codes + d0 / 2) = codes;
            if (d0 % 32 == 0) to[a.exps_at + place * a.row_exps + d0 / 32] = (uint8_t)exp;
            continue;
        }
        if (turns) {
#pragma unroll
            for (int e = 0; e < 8; ++e) own[e] = f32_to_out<BF16>(x[e]);
        }
        if (is_q) {
            if (!known) {
#pragma unroll
                for (int e = 0; e < 8; ++e) own[e] = 0;
            }
            store8<true>(a.q_out + ((int64_t)token * a.q_heads + at) * a.dim + d0, own);
        } else {
            uint8_t* const to = (is_v ? a.v_cache : a.k_cache) + page * a.page_bytes + row * a.row_bytes + at * a.head_bytes;
            store8<VEC>(reinterpret_cast<uint16_t*>(to) + d0, own);
        }
    }
}

struct ReadArgs {
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const int64_t* slots;
    uint16_t* k;
    uint16_t* v;
    int64_t page_bytes, places;
    uint32_t row_codes, row_exps, exps_at;
    int32_t kv_heads, dim, page_size;
};

// Token blockIdx.x: its keys' and values' words of eight codes.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void read_kernel(const ReadArgs a) {
    const int token = blockIdx.x, units = a.dim / 8, items = 2 * a.kv_heads * units;
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
    // vectors of eight: everything aligned, and the mates of eight elements side by side
    const bool vec = (addresses & 15) == 0 && (strides & 7) == 0 && (!turns || a->rot % (a->interleaved ? 8 : 16) == 0);
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
    p.exp_limit = a->dtype == PW4_DTYPE_F16 ? 127 + 13 : 254;
    const int64_t passes = ceil_div(heads, kThreads / (a->head_dim / 8));
    // few tokens: a workgroup a pass over the heads; many: one goes over them all
    const int64_t shares = a->num_tokens * passes <= 8 * device_cus() ? passes : 1;
    const dim3 grid((unsigned)a->num_tokens, (unsigned)std::min<int64_t>(shares, 65535));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    auto run = [&](auto bf16, auto wide) {
        constexpr bool BF16 = decltype(bf16)::value, VEC = decltype(wide)::value;
        if (fp4) {
            hipLaunchKernelGGL((append_kernel<BF16, VEC, true>), grid, dim3(kThreads), 0, s, p);
        } else {
            hipLaunchKernelGGL((append_kernel<BF16, VEC, false>), grid, dim3(kThreads), 0, s, p);
        }
    };
    const auto with_vec = [&](auto bf16) { vec ? run(bf16, std::true_type{}) : run(bf16, std::false_type{}); };
    a->dtype == PW4_DTYPE_BF16 ? with_vec(std::true_type{}) : with_vec(std::false_type{});
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
                     (int32_t)kv_heads, (int32_t)head_dim, (int32_t)page_size};
    const int64_t passes = ceil_div(2 * kv_heads * (head_dim / 8), kThreads);
    const int64_t shares = num_tokens * passes <= 8 * device_cus() ? passes : 1;
    const dim3 grid((unsigned)num_tokens, (unsigned)std::min<int64_t>(shares, 65535));
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

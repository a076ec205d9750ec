// What the attention kernels over paged caches share, whatever the cache holds: a call's
// parameters, the tiles of query rows and their split over workgroups, the parts of a
// softmax, and the writing and joining of results.
//
// A kernel's Keys names how its cache is read one element at a time, for the rows that
// are computed without matrix instructions:
//   element<BF16>(params, plane, kv head, page, row of the page, d)   as fp32
//   kRepeats: a head narrower than the kernel's repeats its elements against zeros
//   kFresh: what depends on the lane alone is computed at the ends of pieces, rather than ahead of them
//     and held in registers through their loops
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdlib>

#include "paged_common.h"
#include "pulsar_paged.h"

namespace pw4 {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* tables;
    const int32_t* lens;
    const int32_t* cu;
    uint16_t* out;
    float* lse;
    float* part_o;    // [2 * workgroups, rows of a tile, dim]
    float* part_ml;   // [2 * workgroups, rows of a tile, 2]: maximum (base 2), sum
    int64_t q_token, q_head, table_stride;            // elements
    uint32_t page_bytes, row_bytes, head_bytes;       // the caches' strides
    int32_t* plan;           // split: what the second launch has to know (PlanOut)
    int32_t num_tokens, batch, q_heads, kv_heads, group, dim, num_pages, page_size;
    int32_t page_shift;      // of a page size that is a power of two, else -1
    uint32_t page_magic;     // else key / page_size = (key * page_magic) >> (32 + page_magic_shift)
    int32_t page_magic_shift;
    int32_t max_q, max_len;  // max_len: keys that tables and caller allow
    int32_t window;
    float scale2;            // |scale| log2(e), above 0; with a cap, scale / cap
    float cap2;              // cap log2(e), 0 without a cap
    uint32_t flip;           // sign bits of q's elements to turn over: a negative scale without a cap
    int32_t flat;            // 2: pages of a power of two of keys, 16 at least; 1: of a multiple of 8
    int32_t min_units;       // split: units (blocks of keys) a workgroup takes at least
    int32_t split;           // 1: runs of units over the grid; 0: a workgroup a tile and head
    int32_t order;           // whole: up to 64 sequences are taken by the lengths of their tiles (Pieces' ORDER)
};

// ---- small device parts ------------------------------------------------------

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)p; }

// One LDS copy instruction: lane l copies 16 (or 4) bytes to LDS[lds + l * 16 (or 4)],
// from its own address, or from a wave-uniform base and its own byte offset.  Issued
// from assembly so that the compiler does not wait for it before LDS reads: the kernels
// count the copies (wait_copies).
__device__ __forceinline__ void lds_copy16(const void* from, uint32_t lds) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(from), "s"(lds)
        : "memory");
}
__device__ __forceinline__ void lds_copy16(const void* base, uint32_t offset, uint32_t lds) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(offset), "s"(base), "s"(lds)
        : "memory");
}
__device__ __forceinline__ void lds_copy4(const void* from, uint32_t lds) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dword %1, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(from), "s"(lds)
        : "memory");
}

// Until at most N of this wave's copies (and older loads) are under way.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N >= 0 && N < 64, "vmcnt is six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ u32x2 read_transposed(const uint8_t* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    using Lds = __attribute__((address_space(3))) s16x4*;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(uintptr_t)(uint32_t)(uintptr_t)p));
}

// A value of lanes l and l ^ 32, in both lanes; or of l and l ^ 16.  (The elements
// are copied out first: a bit cast of a vector's element takes its first one.)
__device__ __forceinline__ f32x2 with_half(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return f32x2{__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)};
}
__device__ __forceinline__ f32x2 with_quarter(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return f32x2{__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)};
}
__device__ __forceinline__ float max_halves(float v) {
    const f32x2 r = with_half(v);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum_halves(float v) {
    const f32x2 r = with_half(v);
    return r[0] + r[1];
}
__device__ __forceinline__ float max_quarters(float v) {
    const f32x2 r = with_quarter(v);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum_quarters(float v) {
    const f32x2 r = with_quarter(v);
    return r[0] + r[1];
}

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t u) {
    if constexpr (BF16) {
        return __builtin_bit_cast(float, (uint32_t)u << 16);
    } else {
        return (float)__builtin_bit_cast(_Float16, u);
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (BF16) {
        return pack_bf16x2_rne(lo, hi);
    } else {
        return as_u32(__builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
}

__device__ __forceinline__ int first_above(const int* ends, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > v) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    return lo;
}

// Scores are held raw, or with a cap as tanh(s scale / cap); their factor `unit()` (to
// units of log2) goes into the exponent's fma.
template <bool CAP>
__device__ __forceinline__ float unit(const Params& a) {
    return CAP ? a.cap2 : a.scale2;
}

// tanh for |x| < kSeries by its Taylor series, within 1.5 * 2^-24 of tanh there before the
// fmas' roundings (the next term): 1 - 2 / (e^2x + 1) subtracts two numbers near 1, so its error is 2^-24 of 1 at
// least, which a cap far above the scores would make an error of 2^-24 of the cap.
constexpr float kSeries = 0.5f;
__device__ __forceinline__ float tanh_series(float x) {
    const float y = x * x;
    float p = 21844.f / 6081075;
    p = __builtin_fmaf(p, y, -1382.f / 155925);
    p = __builtin_fmaf(p, y, 62.f / 2835);
    p = __builtin_fmaf(p, y, -17.f / 315);
    p = __builtin_fmaf(p, y, 2.f / 15);
    p = __builtin_fmaf(p, y, -1.f / 3);
    return __builtin_fmaf(x * y, p, x);
}
// The same in two fmas less: x + x^3 p(x^2), p of degree 3 fitted to the least largest relative error below
// kSeries (Lawson's iteration on 4001 points): the polynomial is within 2^-25.7 of tanh, in fp32 within 1.25 * 2^-24.
__device__ __forceinline__ float tanh_fit(float x) {
    const float y = x * x;
    float p = 0x1.1abd06p-6f;
    p = __builtin_fmaf(p, y, -0x1.b29c18p-5f);
    p = __builtin_fmaf(p, y, 0x1.10ea8ep-3f);
    p = __builtin_fmaf(p, y, -0x1.5554dap-2f);
    return __builtin_fmaf(x * y, p, x);
}
__device__ __forceinline__ float tanh_of(float x) {
    const float e = __builtin_amdgcn_exp2f(x * (2.f * kLog2e));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    return fabsf(x) < kSeries ? tanh_series(x) : far;
}
// With a cap, N raw scores become their tanh.  Every lane of the wave calls it: mostly all
// its scores are far below the cap, and the series is all there is to do.
template <bool CAP, int N, bool FIT = false, typename V>
__device__ __forceinline__ void cap_scores(const Params& a, V& s) {
    if constexpr (CAP) {
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            s[e] *= a.scale2;
            most = fmaxf(most, fabsf(s[e]));
        }
        if (__builtin_expect(__any(most >= kSeries), 0)) {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = tanh_of(s[e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = FIT ? tanh_fit(s[e]) : tanh_series(s[e]);
        }
    }
}

// fp16 probabilities are held times 2^6, so that those of keys far below the
// maximum are not subnormal; the sum is held the same way, so outputs need nothing.
template <bool BF16>
constexpr float kLift = BF16 ? 0.f : 6.f;
// What the exponents are taken against, for a maximum m of raw scores.
template <bool BF16>
__device__ __forceinline__ float shift_of(float m, float k) {
    return __builtin_fmaf(m, k, -kLift<BF16>);
}
// The maximum (units of log2) that a row's sums are held by, to the bit: fp16's shift is rounded
// by up to 2^-22 more than m k, which the lse would take over.
template <bool BF16>
__device__ __forceinline__ float held_max(float m, float k) {
    return shift_of<BF16>(m, k) + kLift<BF16>;
}
// The running maximum is renewed, and sums and outputs scaled, once a score is
// above it by this much (in units of log2): a probability is at most 2^(8 + lift).
constexpr float kSlack = 8.f;

// ---- tiles -------------------------------------------------------------------

// The new tokens of sequence b that are computed, and the keys it has.
struct Sequence {
    int q0, n, first_pos, len;
};
__device__ __forceinline__ Sequence sequence(const Params& a, int b) {
    const int c0 = a.cu[b], c1 = a.cu[b + 1], l = a.lens[b];
    Sequence s;
    s.q0 = min(max(c0, 0), a.num_tokens);
    s.n = min(max(min(c1, a.num_tokens) - s.q0, 0), a.max_q);
    s.first_pos = l - (c1 - c0);
    s.len = min(max(l, 0), a.max_len);
    return s;
}

// The first key that a query at `pos` sees.  (A query before the first key sees none; its window's end, taken as
// that of position 0, stays in 32 bits.)
__device__ __forceinline__ int lowest_key(const Params& a, int pos) {
    return a.window > 0 ? max(0, max(pos, 0) + 1 - a.window) : 0;
}

// A tile: query rows [row0, row0 + rows) of a sequence; keys [lo, hi) are those
// that some row sees, and blocks of keys start at `base`.
struct Tile {
    int b, q0, first_pos, len, row0, rows, lo, hi, base;
};
template <int MR, int KEYS>
__device__ __forceinline__ Tile tile_of(const Params& a, int b, int t, const Sequence& s) {
    Tile r;
    r.b = b;
    r.q0 = s.q0;
    r.first_pos = s.first_pos;
    r.len = s.len;
    r.row0 = t * MR;
    r.rows = min(MR, s.n * a.group - r.row0);
    const int first = s.first_pos + r.row0 / a.group, last = s.first_pos + (r.row0 + max(r.rows, 1) - 1) / a.group;
    r.hi = max(0, min(last + 1, s.len));
    r.lo = lowest_key(a, first);
    if (r.lo >= r.hi) r.lo = r.hi = 0;  // no key
    r.base = r.lo / KEYS * KEYS;
    return r;
}
// Units of UNIT keys; a tile without keys still has one, whose result is empty.
template <int UNIT>
__device__ __forceinline__ int units_of(const Tile& t) {
    return t.rows <= 0 ? 0 : t.hi > t.lo ? (t.hi - t.base + UNIT - 1) / UNIT : 1;
}

constexpr int kMaxSplitTiles = 1024;  // tiles and sequences of a split call

// The units of every tile, ascending sums, in LDS: tiles of sequence b are [seq_end[b - 1], seq_end[b]).
struct Plan {
    int seq_end[kMaxSplitTiles];
    int unit_end[kMaxSplitTiles];
    int scratch[16];
};
// Fills the plan; returns the number of tiles.  Every thread of the workgroup calls it.
template <int MR, int KEYS, int UNIT, int WAVES>
__device__ __forceinline__ int make_plan(const Params& a, Plan& p) {
    int tiles = 0;
    for (int b0 = 0; b0 < a.batch; b0 += WAVES * 64) {
        const int b = b0 + (int)threadIdx.x;
        const int mine = b < a.batch ? (sequence(a, b).n * a.group + MR - 1) / MR : 0;
        int total;
        const int upto = block_inclusive_scan<WAVES>(mine, p.scratch, total);
        if (b < a.batch) p.seq_end[b] = tiles + upto;
        tiles += total;
    }
    tiles = min(tiles, kMaxSplitTiles);
    __syncthreads();
    int units = 0;
    for (int t0 = 0; t0 < tiles; t0 += WAVES * 64) {
        const int t = t0 + (int)threadIdx.x;
        int mine = 0;
        if (t < tiles) {
            const int b = first_above(p.seq_end, a.batch, t);
            mine = units_of<UNIT>(tile_of<MR, KEYS>(a, b, t - (b ? p.seq_end[b - 1] : 0), sequence(a, b)));
        }
        int total;
        const int upto = block_inclusive_scan<WAVES>(mine, p.scratch, total);
        if (t < tiles) p.unit_end[t] = units + upto;
        units += total;
    }
    __syncthreads();
    return tiles;
}

// The units of all tiles and heads, `total` of them, in `parts` runs that differ by one at
// most.  (The host keeps total below 2^31.)
struct Runs {
    int parts, each, more;  // the first `more` runs have each + 1 units
    __device__ __forceinline__ Runs(const Params& a, int total, int grid) {
        parts = max(1, min(grid, total / a.min_units));
        each = total / parts;
        more = total - each * parts;
    }
    __device__ __forceinline__ int begin(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int of(int unit) const {  // the run that a unit is in
        const int longer = more * (each + 1);
        return unit < longer ? unit / (each + 1) : more + (unit - longer) / max(each, 1);
    }
};

// ---- one query row without matrix instructions ---------------------------------

// A wave's pass over keys [begin, end) for one query: for rows that a value which
// is not finite has reached through a key that they do not see (0 * NaN in a
// matrix product).  Lane l holds output elements l, l + 64, ...
struct RowResult {
    float m2, z, o[4];
};
template <typename Keys, bool BF16, bool CAP, typename P>
__device__ __forceinline__ RowResult plain_row(const P& a, int b, int token, int head, int begin, int end) {
    int lane = threadIdx.x & 63;
    if (Keys::kFresh) asm volatile("" : "+v"(lane));
    const int kv = head / a.group;
    const uint16_t* const q = a.q + token * a.q_token + head * a.q_head;
    RowResult r{-kInf, 0.f, {0.f, 0.f, 0.f, 0.f}};
    for (int j0 = begin; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        float s = -kInf;
        uint32_t page = 0, at = 0;  // the lane's key's, and its row there
        if (j < end) {
            page = min((uint32_t)a.tables[b * a.table_stride + j / a.page_size], (uint32_t)a.num_pages - 1);
            at = j % a.page_size;
            float dot = 0.f;
            for (int d = 0; d < a.dim; ++d) dot += to_float<BF16>(q[d]) * Keys::template element<BF16>(a, a.k, kv, page, at, d);
            s = (CAP ? tanh_of(dot * a.scale2) : a.flip ? -dot : dot) * unit<CAP>(a);
        }
        const float m = fmaxf(r.m2, wave_max(s)), shift = m == -kInf ? 0.f : m;
        const float p = __builtin_amdgcn_exp2f(s - shift), scale = __builtin_amdgcn_exp2f(r.m2 - shift);
        r.m2 = m;
        r.z = r.z * scale + wave_sum(p);
        for (int e = 0; e < 4; ++e) r.o[e] *= scale;
        for (int k = 0; k < 64 && j0 + k < end; ++k) {
            const float pk = __shfl(p, k);
            const uint32_t page_k = __shfl(page, k), at_k = __shfl(at, k);
            for (int e = 0; e < 4; ++e) {
                if (lane + 64 * e < a.dim) r.o[e] += pk * Keys::template element<BF16>(a, a.v, kv, page_k, at_k, lane + 64 * e);
            }
        }
    }
    return r;
}

// ---- keys in LDS ---------------------------------------------------------------------

// 16-byte units of a row, and the XOR that places unit c of row r at c ^ swizzle.
// K: the 16 lanes of a phase read one unit of 16 rows.  V: the transposing reads of
// a phase take, of rows that differ in their low bits, 64 bytes of 4 rows (tiles of
// 32 columns, WIDE) or 32 bytes of 8.  Rows of 128 bytes lie two to the 256 of a phase.
template <int DP>
__device__ __forceinline__ int k_swizzle(int r) {
    return DP == 64 ? (r >> 1) & 7 : r & 15;
}
template <int DP, bool WIDE>
__device__ __forceinline__ int v_swizzle(int r) {
    if constexpr (WIDE) return DP == 64 ? ((r >> 1) & 1) * 4 : (r & 3) * 4;
    return DP == 64 ? ((r >> 1) & 3) * 2 : (r & 7) * 2;
}
__device__ __forceinline__ int page_index(const Params& a, int key) {
    return a.page_shift >= 0 ? key >> a.page_shift : (int)(__umulhi((uint32_t)key, a.page_magic) >> a.page_magic_shift);
}

// Query row `row` of the tile as the B operand of K Q^T: 16 bytes of each step of
// the head, from unit `unit` on, `step` units apart; zeros past the head or the tile.
template <int STEPS>
__device__ __forceinline__ void load_query(const Params& a, const Tile& t, int head, int row, int unit, int step,
                                           u32x4 (&q)[STEPS]) {
    const bool in = row < t.rows;
    const int r = t.row0 + min(row, max(t.rows - 1, 0)), i = r / a.group;
    const uint16_t* const from = a.q + (t.q0 + i) * a.q_token + (head * a.group + r - i * a.group) * a.q_head;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int u = unit + s * step;
        q[s] = u32x4{0, 0, 0, 0};
        if (in && u * 8 < a.dim) q[s] = *reinterpret_cast<const u32x4*>(from + u * 8) ^ a.flip;
    }
}

// Whether a value of keys [begin, end) is not finite (a wave's scan).
template <typename Keys, bool BF16, typename P>
__device__ __forceinline__ bool values_not_finite(const P& a, const Tile& t, int head, int begin, int end) {
    bool bad = false;
    for (int key = max(begin, t.lo); key < min(end, t.hi); ++key) {
        const uint32_t page = min((uint32_t)a.tables[t.b * a.table_stride + page_index(a, key)], (uint32_t)a.num_pages - 1);
        const uint32_t at = key - page_index(a, key) * a.page_size;
        int first = threadIdx.x & 63;
        if (Keys::kFresh) asm volatile("" : "+v"(first));
        for (int d = first; d < a.dim; d += 64) {
            const float x = Keys::template element<BF16>(a, a.v, head, page, at, d);
            bad |= x - x != 0.f;
        }
    }
    return __any(bad);
}

// Whether rows whose output is not finite have to be computed again one by one: some
// key of [t.lo, t.hi) that not every row sees has a value that is not finite, or the first or
// the last one has, which stand in for the block's keys outside (a probability of 0, and
// 0 * inf is not inf), or the head is narrower than the kernel's and its padding repeats key
// elements against zeros.
template <typename Keys, bool BF16, typename P>
__device__ __forceinline__ bool must_repeat(const P& a, const Tile& t, int head, int dp) {
    if (Keys::kRepeats && a.dim != dp) return true;
    const int first = t.first_pos + t.row0 / a.group, last = t.first_pos + (t.row0 + t.rows - 1) / a.group;
    if (values_not_finite<Keys, BF16>(a, t, head, min(first + 1, t.hi - 1), t.hi)) return true;
    return a.window > 0 && values_not_finite<Keys, BF16>(a, t, head, t.lo, max(last + 1 - a.window, t.lo + 1));
}

// Where a piece of a tile goes: the call's outputs, or partial slot `slot` >= 0.  (A row whose
// scores are all NaN has a maximum of -inf too, but a sum of NaN, and so has its lse.)
template <int MR, bool BF16>
__device__ __forceinline__ void store_stats(const Params& a, const Tile& t, int head, int row, int slot, float m2, float z) {
    if (slot >= 0) {
        float* const ml = a.part_ml + ((int64_t)slot * MR + row) * 2;
        ml[0] = m2;
        ml[1] = z;
    } else if (a.lse != nullptr) {
        const int r = t.row0 + row, i = r / a.group;
        a.lse[(int64_t)(t.q0 + i) * a.q_heads + head * a.group + r - i * a.group] =
            m2 == -kInf && z == 0.f ? -kInf : (m2 + __builtin_amdgcn_logf(z * (BF16 ? 1.f : 0x1p-6f))) * kLn2;
    }
}
__device__ __forceinline__ uint16_t* out_row(const Params& a, const Tile& t, int head, int row) {
    const int r = t.row0 + row, i = r / a.group;
    return a.out + ((int64_t)(t.q0 + i) * a.q_heads + head * a.group + r - i * a.group) * a.dim;
}

// Tokens begin, begin + step, ... of [begin, end): out 0, lse -inf.
__device__ __forceinline__ void clear_tokens(const Params& a, int begin, int end, int step) {
    const int64_t per_token = (int64_t)a.q_heads * a.dim;
    for (int t = begin; t < end; t += step) {
        for (int64_t e = (int64_t)threadIdx.x * 8; e < per_token; e += blockDim.x * 8) {
            *reinterpret_cast<u32x4*>(a.out + t * per_token + e) = u32x4{0, 0, 0, 0};
        }
        if (a.lse != nullptr) {
            for (int h = threadIdx.x; h < a.q_heads; h += blockDim.x) a.lse[(int64_t)t * a.q_heads + h] = -kInf;
        }
    }
}
// Rows of out that no tile has: past the last sequence, and of each sequence past the
// max_q tokens that are computed (a workgroup a sequence).
__device__ __forceinline__ void clear_rest(const Params& a) {
    const int first = a.batch > 0 ? min(max(a.cu[a.batch], 0), a.num_tokens) : 0;
    if (a.max_q < a.num_tokens) {
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
            const int c0 = min(max(a.cu[b], 0), a.num_tokens), c1 = min(a.cu[b + 1], a.num_tokens);
            if (c1 - c0 > a.max_q) clear_tokens(a, c0 + a.max_q, c1, 1);
        }
    }
    if (first < a.num_tokens) clear_tokens(a, first + (int)blockIdx.x, a.num_tokens, gridDim.x);
}

// What the second launch of a split call reads: the tiles and units there are, then for
// each tile its ascending units and where its rows lie.
struct PlanOut {
    static constexpr int kTiles = 0, kUnits = 1, kEntries = 4;
    struct Entry {
        int begin, end, q0, row0, rows, pad[3];
    };
    static constexpr int kInts = kEntries + 8 * kMaxSplitTiles;
};
__device__ __forceinline__ void write_plan(const Params& a, int i, int begin, int end, const Tile& t) {
    reinterpret_cast<PlanOut::Entry*>(a.plan + PlanOut::kEntries)[i] = PlanOut::Entry{begin, end, t.q0, t.row0, t.rows, {}};
}

// A workgroup's pieces of work, one after the other: units [u0, u1) of a tile and
// head, for partial slot `slot`, or the whole of it (-1).  ONE: a sequence has one tile;
// IN_LDS: those of up to 64 sequences are held in LDS, 64 Tiles at the plan's place, and not in registers.
// ORDER: of whole tiles more than run alone on a CU, the sequences with the longer ones come first, so that
// those that have to share one, or come late, are short.
template <int MR, int KEYS, int UNIT, int WAVES, bool ONE, bool IN_LDS = false, bool ORDER = false>
struct Pieces {
    Tile t;
    int head, u0, u1, slot;
    int at = 0, end = 0, tiles = 0, units = 0, w = 0;
    // ONE, up to 64 sequences: the tile of sequence `lane` and its ascending units, and no plan in LDS
    Tile my;
    int my_end = 0;
    bool fresh = true;

    __device__ __forceinline__ bool in_wave(const Params& a) const { return ONE && a.batch <= 64; }

    __device__ __forceinline__ void set_tile(const Params& a, int b, int place) {
        b = __builtin_amdgcn_readfirstlane(b);
        t = tile_of<MR, KEYS>(a, b, __builtin_amdgcn_readfirstlane(place), sequence(a, b));
        t.q0 = __builtin_amdgcn_readfirstlane(t.q0);
        t.first_pos = __builtin_amdgcn_readfirstlane(t.first_pos);
        t.len = __builtin_amdgcn_readfirstlane(t.len);
        t.row0 = __builtin_amdgcn_readfirstlane(t.row0);
        t.rows = __builtin_amdgcn_readfirstlane(t.rows);
        t.lo = __builtin_amdgcn_readfirstlane(t.lo);
        t.hi = __builtin_amdgcn_readfirstlane(t.hi);
        t.base = __builtin_amdgcn_readfirstlane(t.base);
    }

    // Lane b of a wave has sequence b and its number of tiles: now the sequence that is b-th by its first and
    // last tile's units.
    __device__ __forceinline__ void by_length(const Params& a, int& b, int& n) const {
        int units = 0, place = b;
        if (n > 0) {
            const Sequence s = sequence(a, b);
            units = units_of<KEYS>(tile_of<MR, KEYS>(a, b, 0, s)) + units_of<KEYS>(tile_of<MR, KEYS>(a, b, n - 1, s));
        }
        if (b < a.batch) place = 0;
        for (int other = 0; other < a.batch; ++other) {
            const int theirs = __builtin_amdgcn_readlane(units, other);
            place += b < a.batch && (theirs > units || (theirs == units && other < b));
        }
        n = __builtin_amdgcn_ds_permute(place * 4, n);
        b = __builtin_amdgcn_ds_permute(place * 4, b);
    }

    // Every thread of the workgroup calls these two.
    __device__ __forceinline__ void start(const Params& a, Plan& plan) {
        if (!a.split) return;
        if (in_wave(a)) {
            const int b = threadIdx.x & 63;
            my = Tile{};
            int n = 0;
            if (b < a.batch) {
                my = tile_of<MR, KEYS>(a, b, 0, sequence(a, b));
                n = units_of<UNIT>(my);
            }
            if (IN_LDS) reinterpret_cast<Tile*>(&plan)[b] = my;  // (each wave for itself, and all the same)
            my_end = wave_inclusive_scan(n);
            tiles = a.batch;
            units = __builtin_amdgcn_readlane(my_end, 63);
            if (blockIdx.x == 0 && threadIdx.x < 64 && b < a.batch) write_plan(a, b, my_end - n, my_end, my);
        } else {
            tiles = __builtin_amdgcn_readfirstlane(make_plan<MR, KEYS, UNIT, WAVES>(a, plan));
            units = tiles > 0 ? __builtin_amdgcn_readfirstlane(plan.unit_end[tiles - 1]) : 0;
            if (blockIdx.x == 0) {
                for (int i = threadIdx.x; i < tiles; i += WAVES * 64) {
                    const int b = first_above(plan.seq_end, a.batch, i);
                    const Tile mine = tile_of<MR, KEYS>(a, b, i - (b ? plan.seq_end[b - 1] : 0), sequence(a, b));
                    write_plan(a, i, i ? plan.unit_end[i - 1] : 0, plan.unit_end[i], mine);
                }
            }
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.plan[PlanOut::kTiles] = tiles;
            a.plan[PlanOut::kUnits] = units;
        }
        if (units == 0) return;
        const Runs runs(a, units * a.kv_heads, gridDim.x);
        // runs side by side on one XCD: workgroups go to the XCDs in turn
        w = gridDim.x % 8 == 0 ? (int)(blockIdx.x % 8) * ((int)gridDim.x / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
        if (w >= runs.parts) return;
        at = __builtin_amdgcn_readfirstlane(runs.begin(w));
        end = __builtin_amdgcn_readfirstlane(runs.begin(w + 1));
    }
    __device__ __forceinline__ bool next(const Params& a, const Plan& plan) {
        if (!a.split) {  // tile blockIdx / heads, counted over the sequences, a sequence's last first
            if (!fresh) return false;
            fresh = false;
            head = blockIdx.x % a.kv_heads;
            const int rank = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63;
            u0 = 0;
            slot = -1;
            if (ONE) {  // the rank is the sequence
                if (rank >= a.batch) return false;
                set_tile(a, rank, 0);
                u1 = units_of<UNIT>(t);
                return t.rows > 0;
            }
            int before = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 64) {
                int b = b0 + lane;
                int mine = b < a.batch ? (sequence(a, b).n * a.group + MR - 1) / MR : 0;
                if (ORDER && a.order) by_length(a, b, mine);
                const int upto = before + wave_inclusive_scan(mine);
                const uint64_t past = __ballot(upto > rank);
                if (past != 0) {
                    const int l = __builtin_ctzll(past);
                    set_tile(a, __builtin_amdgcn_readlane(b, l), __builtin_amdgcn_readlane(upto, l) - 1 - rank);
                    u1 = units_of<UNIT>(t);
                    return true;
                }
                before = __builtin_amdgcn_readlane(upto, 63);
            }
            return false;
        }
        if (at >= end) return false;
        head = __builtin_amdgcn_readfirstlane(at / units);
        const int r = at - head * units;
        int first, last;
        if (in_wave(a)) {
            const int b = __builtin_ctzll(__ballot(my_end > r));
            first = b ? __builtin_amdgcn_readlane(my_end, b - 1) : 0;
            last = __builtin_amdgcn_readlane(my_end, b);
            const Tile held = IN_LDS ? reinterpret_cast<const Tile*>(&plan)[b] : my;
            const auto of_b = [&](int v) { return IN_LDS ? __builtin_amdgcn_readfirstlane(v) : __builtin_amdgcn_readlane(v, b); };
            t.b = b;
            t.q0 = of_b(held.q0);
            t.first_pos = of_b(held.first_pos);
            t.len = of_b(held.len);
            t.row0 = 0;
            t.rows = of_b(held.rows);
            t.lo = of_b(held.lo);
            t.hi = of_b(held.hi);
            t.base = of_b(held.base);
        } else {
            const int ti = __builtin_amdgcn_readfirstlane(first_above(plan.unit_end, tiles, r));
            const int b = __builtin_amdgcn_readfirstlane(first_above(plan.seq_end, a.batch, ti));
            first = ti ? plan.unit_end[ti - 1] : 0;
            last = plan.unit_end[ti];
            set_tile(a, b, ti - (b ? plan.seq_end[b - 1] : 0));
        }
        const int all = last - first;
        u0 = __builtin_amdgcn_readfirstlane(r - first);
        u1 = __builtin_amdgcn_readfirstlane(min(all, u0 + (end - at)));
        slot = __builtin_amdgcn_readfirstlane(u0 == 0 && u1 == all ? -1 : 2 * w + (u0 == 0 ? 1 : 0));
        at += u1 - u0;
        return true;
    }
};

// ---- ends of pieces --------------------------------------------------------------------

// The waves of a few-rows workgroup, each with keys of its own, join in LDS: rows of DP + 4
// floats (maximum, sum behind the outputs) from `smem` on.  o[mt][d] holds elements 16 d + 4 g
// .. + 3 of row 16 mt + c, m its maximum, z the lane's share of its sum, over keys [begin, end).  PARTS: the rows
// go through LDS in so many parts, in as much less of it.
template <typename Keys, bool BF16, int DP, int MT, int WAVES, bool CAP, int PARTS = 1, typename P>
__device__ __forceinline__ void join_waves(const P& a, const Tile& t, uint8_t* smem, int wave, int head, int slot, int begin,
                                           int end, float k, const float (&m)[MT], const float (&z)[MT],
                                           const f32x4 (&o)[MT][DP / 16]) {
    constexpr int MR = 16 * MT, DT = DP / 16, PR = MR / PARTS;
    static_assert(MT % PARTS == 0, "whole tiles of 16 rows");
    int lane = threadIdx.x & 63;
    if (Keys::kFresh) asm volatile("" : "+v"(lane));
    const int c = lane & 15, g = lane >> 4;
    constexpr int kRow = DP + 4;
    float* const join = reinterpret_cast<float*>(smem);
    bool bad = false;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        if (part > 0) __syncthreads();
#pragma unroll
        for (int mt = part * MT / PARTS; mt < (part + 1) * MT / PARTS; ++mt) {
            float* const row = join + (wave * PR + mt * 16 - part * PR + c) * kRow;
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(row + d * 16 + 4 * g) = o[mt][d];
            const float all = sum_halves(sum_quarters(z[mt]));
            if (g == 0) {
                row[DP] = held_max<BF16>(m[mt], k);
                row[DP + 1] = all;
            }
        }
        __syncthreads();
        for (int row = part * PR + wave; row < min(t.rows, (part + 1) * PR); row += WAVES) {
            const float* const of_row = join + (row - part * PR) * kRow;  // wave v's is v * PR rows on
            float m2 = -kInf, sum = 0.f, w[WAVES];
#pragma unroll
            for (int v = 0; v < WAVES; ++v) m2 = fmaxf(m2, of_row[v * PR * kRow + DP]);
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const float mv = of_row[v * PR * kRow + DP];
                w[v] = mv == -kInf ? 0.f : __builtin_amdgcn_exp2f(mv - m2);
                sum += w[v] * of_row[v * PR * kRow + DP + 1];
            }
            const float inv = slot >= 0 ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
            uint16_t* const to = slot >= 0 ? nullptr : out_row(a, t, head, row);
            for (int d = lane; d < a.dim; d += 64) {
                float x = 0.f;
#pragma unroll
                for (int v = 0; v < WAVES; ++v) {
                    if (w[v] != 0.f) x += w[v] * of_row[v * PR * kRow + d];
                }
                bad |= x - x != 0.f;
                if (slot >= 0) {
                    a.part_o[((int64_t)slot * MR + row) * a.dim + d] = x;
                } else {
                    to[d] = f32_to_out<BF16>(x * inv);
                }
            }
            if (lane == 0) store_stats<MR, BF16>(a, t, head, row, slot, m2, sum);
            bad |= sum - sum != 0.f;
        }
    }
    if (__any(bad) && must_repeat<Keys, BF16>(a, t, head, DP)) {
        for (int row = wave; row < t.rows; row += WAVES) {
            const int r = t.row0 + row, i = r / a.group, pos = t.first_pos + i;
            const int from = max(begin, a.window > 0 ? pos + 1 - a.window : 0), to = min(end, pos + 1);
            const RowResult x = plain_row<Keys, BF16, CAP>(a, t.b, t.q0 + i, head * a.group + r - i * a.group, max(from, 0), to);
            const float lift = __builtin_amdgcn_exp2f(kLift<BF16>);
            for (int e = 0; e < 4; ++e) {
                const int d = lane + 64 * e;
                if (d >= a.dim) continue;
                if (slot >= 0) {
                    a.part_o[((int64_t)slot * MR + row) * a.dim + d] = x.o[e] * lift;
                } else {
                    out_row(a, t, head, row)[d] = f32_to_out<BF16>(x.z == 0.f ? 0.f : x.o[e] / x.z);
                }
            }
            if (lane == 0) store_stats<MR, BF16>(a, t, head, row, slot, x.m2, x.z * lift);
        }
    }
}

constexpr int kManyKeys = 64;  // keys of a block that a workgroup shares

// A wave's 32 rows of a tile, a row a lane (and the lane 32 from it).
template <int KEYS>
struct WaveRows {
    Tile mine;             // the rows, and the keys that some of them see
    int all_lo, all_hi;    // keys that all of them see
    int row_lo, row_hi;    // keys that the lane's row sees
    __device__ __forceinline__ WaveRows(const Params& a, const Tile& t, int wave) : mine(t) {
        mine.row0 = t.row0 + wave * 32;
        mine.rows = max(0, min(32, t.rows - wave * 32));
        const int pos0 = t.first_pos + mine.row0 / a.group;
        const int pos1 = t.first_pos + (mine.row0 + max(mine.rows, 1) - 1) / a.group;
        const int pos = t.first_pos + (mine.row0 + (int)(threadIdx.x & 31)) / a.group;
        mine.hi = mine.rows > 0 ? max(0, min(pos1 + 1, t.hi)) : 0;
        mine.lo = lowest_key(a, pos0);
        all_hi = min(pos0 + 1, t.hi);
        all_lo = a.window > 0 ? pos1 + 1 - a.window : 0;
        row_hi = min(pos + 1, t.hi);
        row_lo = a.window > 0 ? pos + 1 - a.window : 0;
    }
    // Whether some row sees a key of the block from key0 on.
    __device__ __forceinline__ bool sees(int key0) const { return key0 < mine.hi && key0 + KEYS > mine.lo; }
    // Scores of keys that the lane's row does not see become -inf: s[kt][e] is key 32 kt +
    // 8 (e / 4) + 4 h + e % 4 of the block.
    __device__ __forceinline__ void mask(int key0, int h, f32x16 (&s)[2]) const {
        if (key0 >= all_lo && key0 + KEYS <= all_hi) return;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = key0 + kt * 32 + 8 * (e / 4) + 4 * h + e % 4;
                s[kt][e] = ((key < row_lo) | (key >= row_hi)) ? -kInf : s[kt][e];
            }
    }
};

// The end of a wave's rows: o[d][e] is element 32 d + 8 (e / 4) + 4 h + e % 4 of the lane's row,
// m its maximum in units of log2, z the lane's half of its sum, over keys [begin, end).
template <typename Keys, bool BF16, int DP, int MR, bool CAP, typename P>
__device__ __forceinline__ void store_rows(const P& a, const Tile& t, const WaveRows<kManyKeys>& r, int wave, int head,
                                           int slot, int begin, int end, float m, float z, const f32x16 (&o)[DP / 32]) {
    constexpr int DT = DP / 32;
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    z = sum_halves(z);
    const bool in = c < r.mine.rows;
    const float inv = slot >= 0 ? 1.f : z > 0.f ? 1.f / z : z == 0.f ? 0.f : z;
    bool bad = z - z != 0.f;
    float* const part = slot >= 0 ? a.part_o + ((int64_t)slot * MR + wave * 32 + c) * a.dim : nullptr;
    uint16_t* const to = slot >= 0 || !in ? nullptr : out_row(a, r.mine, head, c);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
            const int at = d * 32 + e4 * 8 + h * 4;
            const f32x4 x{o[d][4 * e4], o[d][4 * e4 + 1], o[d][4 * e4 + 2], o[d][4 * e4 + 3]};
            if (!in || at >= a.dim) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= x[e] - x[e] != 0.f;
            if (slot >= 0) {
                *reinterpret_cast<f32x4*>(part + at) = x;
            } else {
                *reinterpret_cast<u32x2*>(to + at) = u32x2{pack2<BF16>(x[0] * inv, x[1] * inv), pack2<BF16>(x[2] * inv, x[3] * inv)};
            }
        }
    }
    if (in && h == 0) {
        if (slot >= 0) {
            store_stats<MR, BF16>(a, t, head, wave * 32 + c, slot, m, z);
        } else {
            store_stats<MR, BF16>(a, r.mine, head, c, slot, m, z);
        }
    }
    Tile met = r.mine;  // the keys that its products met: whole blocks
    met.lo = max(t.lo, r.mine.lo - (kManyKeys - 1));
    met.hi = min(t.hi, r.mine.hi + (kManyKeys - 1));
    if (__any(in && bad) && must_repeat<Keys, BF16>(a, met, head, DP)) {
        const float lift = __builtin_amdgcn_exp2f(kLift<BF16>);
        for (int row = 0; row < r.mine.rows; ++row) {
            const int at_row = r.mine.row0 + row, i = at_row / a.group, at = t.first_pos + i;
            const int from = max(begin, a.window > 0 ? at + 1 - a.window : 0);
            const RowResult x = plain_row<Keys, BF16, CAP>(a, t.b, t.q0 + i, head * a.group + at_row - i * a.group, from, min(end, at + 1));
            for (int e = 0; e < 4; ++e) {
                const int d = lane + 64 * e;
                if (d >= a.dim) continue;
                if (slot >= 0) {
                    a.part_o[((int64_t)slot * MR + wave * 32 + row) * a.dim + d] = x.o[e] * lift;
                } else {
                    out_row(a, r.mine, head, row)[d] = f32_to_out<BF16>(x.z == 0.f ? 0.f : x.o[e] / x.z);
                }
            }
            if (lane == 0) store_stats<MR, BF16>(a, slot >= 0 ? t : r.mine, head, slot >= 0 ? wave * 32 + row : row, slot, x.m2, x.z * lift);
        }
    }
}

// ---- joining partial results --------------------------------------------------------

// Row blockIdx.y * 4 + wave of tile and head blockIdx.x, a wave a row.
template <int MR, bool BF16>
__global__ __launch_bounds__(256) void join_kernel(const Params a, int grid) {
    const int ti = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads;
    const int row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const PlanOut::Entry e = reinterpret_cast<const PlanOut::Entry*>(a.plan + PlanOut::kEntries)[ti];
    const int units = a.plan[PlanOut::kUnits];
    if (ti >= a.plan[PlanOut::kTiles] || row >= e.rows || e.end <= e.begin) return;
    const Runs runs(a, units * a.kv_heads, grid);
    const int w0 = runs.of(head * units + e.begin), n = runs.of(head * units + e.end - 1) - w0 + 1;
    if (n == 1) return;
    // partial i: the first run's second slot, then the others' first ones
    const auto slot = [&](int i) -> int64_t { return 2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0); };
    float m2 = -kInf;
    for (int i = lane; i < n; i += 64) m2 = fmaxf(m2, a.part_ml[(slot(i) * MR + row) * 2]);
    m2 = wave_max(m2);
    constexpr int kAtOnce = 8;
    float z = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n; i0 += 64) {
        float w = 0.f;
        if (i0 + lane < n) {
            const float* const ml = a.part_ml + (slot(i0 + lane) * MR + row) * 2;
            w = ml[0] == -kInf ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m2);
            z += ml[0] == -kInf && ml[1] == 0.f ? 0.f : w * ml[1];
        }
        const int here = min(64, n - i0);
        for (int i = 0; i < here; i += kAtOnce) {  // so many loads under way
            float v[kAtOnce][4];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float* const o = a.part_o + (slot(i0 + min(i + u, here - 1)) * MR + row) * a.dim;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[u][j] = lane + 64 * j < a.dim ? o[lane + 64 * j] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float wi = __shfl(w, min(i + u, 63));  // 0 past the last
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] += wi == 0.f ? 0.f : wi * v[u][j];  // a run of no weight may hold anything
            }
        }
    }
    z = wave_sum(z);
    const float inv = z > 0.f ? 1.f / z : z == 0.f ? 0.f : z;
    Tile t{};
    t.q0 = e.q0;
    t.row0 = e.row0;
    uint16_t* const to = out_row(a, t, head, row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (lane + 64 * j < a.dim) to[lane + 64 * j] = f32_to_out<BF16>(x[j] * inv);
    }
    if (lane == 0) store_stats<MR, BF16>(a, t, head, row, -1, m2, z);
}

// The same with a workgroup a row (blockIdx.y), whose waves take the partials in turn: for few rows in
// many pieces.
template <int MR, bool BF16, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void join_row_kernel(const Params a, int grid) {
    constexpr int kAtOnce = 8;
    __shared__ float s_x[WAVES][256], s_ml[WAVES][2];
    const int ti = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads, row = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PlanOut::Entry e = reinterpret_cast<const PlanOut::Entry*>(a.plan + PlanOut::kEntries)[ti];
    const int units = a.plan[PlanOut::kUnits];
    if (ti >= a.plan[PlanOut::kTiles] || row >= e.rows || e.end <= e.begin) return;
    const Runs runs(a, units * a.kv_heads, grid);
    const int w0 = runs.of(head * units + e.begin), n = runs.of(head * units + e.end - 1) - w0 + 1;
    if (n == 1) return;
    // partial i: the first run's second slot, then the others' first ones
    const auto slot = [&](int i) -> int64_t { return 2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0); };
    float m2 = -kInf, z = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = wave * kAtOnce; i0 < n; i0 += WAVES * kAtOnce) {
        float v[kAtOnce][4], m[kAtOnce], l[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t at = slot(min(i0 + u, n - 1)) * MR + row;
            m[u] = i0 + u < n ? a.part_ml[at * 2] : -kInf;
            l[u] = i0 + u < n ? a.part_ml[at * 2 + 1] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = lane + 64 * j < a.dim ? a.part_o[at * a.dim + lane + 64 * j] : 0.f;
        }
        float top = m2;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, m[u]);
        const float scale = m2 == -kInf ? 0.f : __builtin_amdgcn_exp2f(m2 - top);
        z = z == 0.f ? 0.f : z * scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = scale == 0.f ? 0.f : x[j] * scale;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const float w = m[u] == -kInf ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
            z += m[u] == -kInf && l[u] == 0.f ? 0.f : m[u] == -kInf ? l[u] - l[u] : w * l[u];  // a sum of NaN has a maximum of -inf
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] += w == 0.f ? 0.f : w * v[u][j];  // a run of no weight may hold anything
        }
        m2 = top;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s_x[wave][lane + 64 * j] = x[j];
    if (lane == 0) {
        s_ml[wave][0] = m2;
        s_ml[wave][1] = z;
    }
    __syncthreads();
    if (wave != 0) return;
    m2 = -kInf;
    z = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m2 = fmaxf(m2, s_ml[w][0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float f = s_ml[w][0] == -kInf ? 0.f : __builtin_amdgcn_exp2f(s_ml[w][0] - m2);
        z += s_ml[w][0] == -kInf ? s_ml[w][1] : f * s_ml[w][1];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += f == 0.f ? 0.f : f * s_x[w][lane + 64 * j];
    }
    const float inv = z > 0.f ? 1.f / z : z == 0.f ? 0.f : z;
    Tile t{};
    t.q0 = e.q0;
    t.row0 = e.row0;
    uint16_t* const to = out_row(a, t, head, row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (lane + 64 * j < a.dim) to[lane + 64 * j] = f32_to_out<BF16>(x[j] * inv);
    }
    if (lane == 0) store_stats<MR, BF16>(a, t, head, row, -1, m2, z);
}

// ---- host ----------------------------------------------------------------------------

inline int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// The parameters but for the caches' strides and the split.  `a` has passed its check.
inline Params params_of(const pw4_paged_attention_args* a) {
    Params p{};
    p.q = static_cast<const uint16_t*>(a->q);
    p.k = static_cast<const uint16_t*>(a->k_cache);
    p.v = static_cast<const uint16_t*>(a->v_cache);
    p.tables = a->block_tables;
    p.lens = a->seq_lens;
    p.cu = a->cu_q;
    p.out = static_cast<uint16_t*>(a->out);
    p.lse = a->lse;
    p.q_token = a->q_token_stride;
    p.q_head = a->q_head_stride;
    p.table_stride = a->table_stride;
    p.num_tokens = (int32_t)a->num_tokens;
    p.batch = (int32_t)a->batch;
    p.q_heads = (int32_t)a->q_heads;
    p.kv_heads = (int32_t)a->kv_heads;
    p.group = (int32_t)(a->q_heads / a->kv_heads);
    p.dim = (int32_t)a->head_dim;
    p.num_pages = (int32_t)a->num_pages;
    p.page_size = (int32_t)a->page_size;
    p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? __builtin_ctzll((uint64_t)a->page_size) : -1;
    if (p.page_shift < 0) {  // 2^(31 + s) / size, rounded up, for 2^(s - 1) < size < 2^s: exact for keys below 2^31
        const int bits = 64 - __builtin_clzll((uint64_t)a->page_size);
        p.page_magic = (uint32_t)(((1ull << (31 + bits)) + a->page_size - 1) / a->page_size);
        p.page_magic_shift = bits - 1;
    }
    p.max_q = (int32_t)std::min(a->max_q_len, a->num_tokens);
    const int64_t held = a->num_pages == 0 ? 0 : std::min<int64_t>(INT_MAX, a->table_width * a->page_size);
    p.max_len = (int32_t)std::min(a->max_seq_len, held);
    p.window = (int32_t)a->window;
    // a scale of 0 is held as one that leaves nothing of a score either, so that -inf stays -inf
    // Caps are held between 2^-100 and 2^100: no e^s tells a smaller one from 0, and what a
    // larger one takes off a score below 2^88 is lost in the score's own rounding.
    const float cap = std::min(std::max(a->softcap, 0x1p-100f), 0x1p100f);
    p.scale2 = a->softcap > 0.f ? std::min(std::max(a->scale / cap, -FLT_MAX), FLT_MAX)
                                : std::max(std::fabs(a->scale) * kLog2e, 0x1p-100f);
    p.flip = a->softcap > 0.f || a->scale >= 0.f ? 0 : 0x80008000u;
    p.cap2 = a->softcap > 0.f ? cap * kLog2e : 0.f;
    return p;
}

// Whether a launch may have so many workgroups: the device counts threads in 32 bits, and runs what is left of
// the count without an error.
inline bool fits_a_launch(int64_t groups, int waves) { return groups <= UINT32_MAX / (waves * 64); }

// Runs a kernel with more LDS than a kernel may have unasked; the permission is
// asked for once a kernel and device.  `plan`: bytes behind its stages, a Plan's at most.
template <auto Kernel, typename P>
hipError_t run_attention(const P& p, int grid, int waves, int stages, int plan, hipStream_t s) {
    const int most = stages + (int)sizeof(Plan), lds = stages + plan;
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
    if (dev < 0 || dev >= 64 || (allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != hipSuccess) return e;
        if (dev >= 0 && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(Kernel, dim3((unsigned)std::max(grid, 1)), dim3(waves * 64), lds, s, p);
    return hipGetLastError();
}

// The second launch of a split call whose first one had `grid` workgroups.
template <int MR, bool BF16>
void run_join(const Params& p, int64_t tiles, int grid, hipStream_t s) {
    hipLaunchKernelGGL((join_kernel<MR, BF16>), dim3((unsigned)(tiles * p.kv_heads), MR / 4), dim3(256), 0, s, p, grid);
}

template <int MR, bool BF16, int WAVES>
void run_row_join(const Params& p, int64_t tiles, int rows, int grid, hipStream_t s) {
    hipLaunchKernelGGL((join_row_kernel<MR, BF16, WAVES>), dim3((unsigned)(tiles * p.kv_heads), rows), dim3(WAVES * 64), 0, s,
                       p, grid);
}

// The workspace of a split call: partial outputs, their maxima and sums, and the plan.
inline size_t partial_bytes(int64_t grid, int64_t tile_rows, int64_t dim) {
    return (size_t)(2 * grid * tile_rows * (dim + 2) + PlanOut::kInts) * 4;
}
inline void place_partials(Params& p, void* workspace, int64_t grid, int64_t tile_rows) {
    const int64_t rows = 2 * grid * tile_rows;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + rows * p.dim;
    p.plan = reinterpret_cast<int32_t*>(p.part_ml + rows * 2);
}

// What holds for any cache: the checks of a call's arguments but for the caches' strides.
inline int check_attention(const pw4_paged_attention_args* a) {
    if (a == nullptr) return PW4_ERR_ARG;
    if (a->dtype != PW4_DTYPE_F16 && a->dtype != PW4_DTYPE_BF16) return PW4_ERR_ARG;
    for (int64_t v : {a->num_tokens, a->batch, a->num_pages, a->table_width, a->max_q_len, a->max_seq_len, a->window}) {
        if (v < 0) return PW4_ERR_ARG;
        if (v > INT_MAX) return PW4_ERR_SHAPE;
    }
    if (a->q_heads <= 0 || a->kv_heads <= 0 || a->page_size <= 0) return PW4_ERR_ARG;
    if (a->q_heads % a->kv_heads != 0 || a->q_heads > 65535 || a->head_dim <= 0 || a->head_dim > 256 ||
        a->head_dim % 8 != 0 || a->page_size > INT_MAX || a->table_stride < a->table_width) {
        return PW4_ERR_SHAPE;
    }
    // rows of a sequence are counted in 32 bits
    if (std::min(a->max_q_len, a->num_tokens) * (a->q_heads / a->kv_heads) > INT_MAX - 1024) return PW4_ERR_SHAPE;
    if (!(a->softcap >= 0.f) || !std::isfinite(a->softcap) || !std::isfinite(a->scale)) return PW4_ERR_ARG;
    if (a->num_tokens == 0) return PW4_OK;
    if (!a->q || !a->out || !a->cu_q || (a->batch && !a->seq_lens)) return PW4_ERR_ARG;
    if (a->batch && a->table_width && a->num_pages && (!a->k_cache || !a->v_cache || !a->block_tables)) return PW4_ERR_ARG;
    return PW4_OK;
}

}  // namespace
}  // namespace pw4

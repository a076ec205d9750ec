// Attention of new tokens over a paged cache (the definition: pulsar_paged.h).
//
// Rows.  The `group` query heads that share a key-value head and the new tokens
// of a sequence make one matrix of n * group query rows (token-major) against
// the same keys, so one token's group is already a matrix product.  A tile is up
// to 16 (32) rows of a few-rows call, one tile a sequence, or 128 rows else.
//
// Transposed products.  Scores are computed as S^T = K Q^T and outputs as
// O^T = V^T P^T: in the MFMA result layout a lane then holds scores of one query
// row only, so the running maximum and sum of the softmax are a lane's own (and
// one or two half-wave exchanges), and the scores a lane holds are, rounded, the
// very P^T operand that it has to supply next -- nothing goes through LDS.  K
// rows are the A operand as they lie; V^T is read by the transposing LDS loads.
//
// Keys reach LDS by direct copies (no registers), each lane naming its own
// source address, so a page may end anywhere.  Page ids come the same way, two
// blocks ahead.  LDS rows are XOR-swizzled in 16-byte units by permuting the
// source, so that K's ds_read_b128 and V's transposing reads spread over the
// banks.  A key index outside what some row of the tile sees is clamped to one
// that is seen: what lies in unused slots is never read, and masked scores meet
// only values of seen keys.
//
// Splitting.  Where tiles are few, the blocks of keys of all tiles and heads are
// laid end to end and dealt to the workgroups in equal runs, whatever the
// lengths; a tile that falls to several is joined by a second launch from fp32
// partial outputs with their maxima and sums.
#include "pulsar_paged.h"

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdlib>

#include "paged_common.h"

using namespace pw4;

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

// tanh for |x| < kSeries by its Taylor series, the next term of which is below 2^-24 x
// there: 1 - 2 / (e^2x + 1) subtracts two numbers near 1, so its error is 2^-24 of 1 at
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
__device__ __forceinline__ float tanh_of(float x) {
    const float e = __builtin_amdgcn_exp2f(x * (2.f * kLog2e));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    return fabsf(x) < kSeries ? tanh_series(x) : far;
}
// With a cap, N raw scores become their tanh.  Every lane of the wave calls it: mostly all
// its scores are far below the cap, and the series is all there is to do.
template <bool CAP, int N, typename V>
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
            for (int e = 0; e < N; ++e) s[e] = tanh_series(s[e]);
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
    r.lo = a.window > 0 ? max(0, first + 1 - a.window) : 0;
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
template <bool BF16, bool CAP>
__device__ __forceinline__ RowResult plain_row(const Params& a, int b, int token, int head, int begin, int end) {
    const int lane = threadIdx.x & 63;
    const uint64_t kv = (uint64_t)(head / a.group) * a.head_bytes;
    const uint16_t* const q = a.q + token * a.q_token + head * a.q_head;
    RowResult r{-kInf, 0.f, {0.f, 0.f, 0.f, 0.f}};
    for (int j0 = begin; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        float s = -kInf;
        uint64_t at = 0;  // bytes
        if (j < end) {
            const uint32_t page = min((uint32_t)a.tables[b * a.table_stride + j / a.page_size], (uint32_t)a.num_pages - 1);
            at = (uint64_t)page * a.page_bytes + (uint64_t)(j % a.page_size) * a.row_bytes + kv;
            const uint16_t* const key = reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(a.k) + at);
            float dot = 0.f;
            for (int d = 0; d < a.dim; ++d) dot += to_float<BF16>(q[d]) * to_float<BF16>(key[d]);
            s = (CAP ? tanh_of(dot * a.scale2) : a.flip ? -dot : dot) * unit<CAP>(a);
        }
        const float m = fmaxf(r.m2, wave_max(s)), shift = m == -kInf ? 0.f : m;
        const float p = __builtin_amdgcn_exp2f(s - shift), scale = __builtin_amdgcn_exp2f(r.m2 - shift);
        r.m2 = m;
        r.z = r.z * scale + wave_sum(p);
        for (int e = 0; e < 4; ++e) r.o[e] *= scale;
        for (int k = 0; k < 64 && j0 + k < end; ++k) {
            const float pk = __shfl(p, k);
            const uint16_t* const value = reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(a.v) +
                                                                            __shfl((unsigned long long)at, k));
            for (int e = 0; e < 4; ++e) {
                if (lane + 64 * e < a.dim) r.o[e] += pk * to_float<BF16>(value[lane + 64 * e]);
            }
        }
    }
    return r;
}

// ---- copying a block of keys into LDS --------------------------------------------

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

// Where a tile's keys are.
struct Source {
    const uint8_t* k;        // of the key-value head
    const uint8_t* v;
    const int32_t* table;    // the sequence's row
    uint32_t pages1;         // pages - 1
    int lo, last;            // keys are clamped to [lo, last]
};
__device__ __forceinline__ Source source_of(const Params& a, const Tile& t, int head) {
    const uint64_t at = (uint64_t)head * a.head_bytes;
    return Source{reinterpret_cast<const uint8_t*>(a.k) + at, reinterpret_cast<const uint8_t*>(a.v) + at,
                  a.tables + t.b * a.table_stride, (uint32_t)a.num_pages - 1, t.lo, t.hi - 1};
}
__device__ __forceinline__ int clamp_key(const Source& s, int key) { return min(max(key, s.lo), s.last); }
__device__ __forceinline__ int page_index(const Params& a, int key) {
    return a.page_shift >= 0 ? key >> a.page_shift : (int)(__umulhi((uint32_t)key, a.page_magic) >> a.page_magic_shift);
}

// The lane's key's page id into LDS[lds + 4 lane].
__device__ __forceinline__ void copy_pages(const Params& a, const Source& s, int key, uint32_t lds) {
    lds_copy4(s.table + page_index(a, clamp_key(s, key)), lds);
}

// What a lane's 16-byte units of a key's row are, for 16 keys whose first row in the
// stage is a multiple of 16: byte offsets from the 16 keys' first row.
template <int DP>
struct Lanes {
    static constexpr int kUnits = DP / 8, kPer = 64 / kUnits, kSteps = 16 / kPer;  // rows an instruction
    uint32_t at[kSteps];
};
template <int DP, typename F>
__device__ __forceinline__ Lanes<DP> lanes_of(const Params& a, F swizzle) {
    Lanes<DP> l;
    const int lane = threadIdx.x & 63, sub = lane / Lanes<DP>::kUnits, c = lane % Lanes<DP>::kUnits, valid = a.dim / 8;
#pragma unroll
    for (int i = 0; i < Lanes<DP>::kSteps; ++i) {
        const int r = i * Lanes<DP>::kPer + sub;
        int unit = c ^ swizzle(r);
        if (DP / 8 != valid && unit >= valid) unit %= valid;  // a narrower head: its units again
        l.at[i] = (uint32_t)r * a.row_bytes + unit * 16;
    }
    return l;
}

// 16 keys from `first` on (a multiple of 16).  Where they lie in one page and all are seen,
// the byte offset of the first one's row (uniform), `id` being its page's, is all there is
// to find out.
__device__ __forceinline__ bool all_seen(const Source& s, int first) { return first >= s.lo && first + 15 <= s.last; }
__device__ __forceinline__ bool in_one_page(const Params& a, const Source& s, int first) {
    return a.flat == 2 && all_seen(s, first);
}
__device__ __forceinline__ uint64_t row_of(const Params& a, const Source& s, int first, int id) {
    const uint32_t page = min((uint32_t)__builtin_amdgcn_readfirstlane(id), s.pages1);
    return (uint64_t)page * a.page_bytes + (uint32_t)(first & (a.page_size - 1)) * a.row_bytes;
}
// A plane's rows of 16 keys to LDS[to], from the common row `base`.
template <int DP>
__device__ __forceinline__ void copy_rows(const uint8_t* base, const Lanes<DP>& l, uint32_t to) {
#pragma unroll
    for (int i = 0; i < Lanes<DP>::kSteps; ++i) lds_copy16(base, l.at[i], to + i * 1024);
}
// One or two planes' rows of 16 keys that lie in several pages or are not all seen, `ids`
// being the keys' page ids in LDS: an instruction's rows from their common page (pages of
// multiples of 8 keys; an instruction takes 8, 4 or 2), or each lane's from its own.
template <int DP, bool BOTH>
__device__ __forceinline__ void copy_rows_apart(const Params& a, const Source& s, const uint8_t* plane, const Lanes<DP>& l,
                                                uint32_t to, const uint8_t* plane2, const Lanes<DP>& l2, uint32_t to2,
                                                int first, const int* ids) {
    constexpr int PER = Lanes<DP>::kPer;
    if (a.flat && all_seen(s, first)) {
#pragma unroll
        for (int i = 0; i < Lanes<DP>::kSteps; ++i) {
            const int key = first + i * PER;
            const uint32_t page = min((uint32_t)__builtin_amdgcn_readfirstlane(ids[i * PER]), s.pages1);
            const uint32_t in_page = key - page_index(a, key) * a.page_size;
            const uint64_t at = (uint64_t)page * a.page_bytes + in_page * a.row_bytes - (uint64_t)(i * PER) * a.row_bytes;
            lds_copy16(plane + at, l.at[i], to + i * 1024);
            if (BOTH) lds_copy16(plane2 + at, l2.at[i], to2 + i * 1024);
        }
        return;
    }
    const int sub = (threadIdx.x & 63) / Lanes<DP>::kUnits;
#pragma unroll
    for (int i = 0; i < Lanes<DP>::kSteps; ++i) {
        const int r = i * PER + sub, key = clamp_key(s, first + r);
        const uint32_t page = min((uint32_t)ids[r], s.pages1), in_page = key - page_index(a, key) * a.page_size;
        const uint64_t at = (uint64_t)page * a.page_bytes + (uint64_t)in_page * a.row_bytes - (uint32_t)r * a.row_bytes;
        lds_copy16(plane + at + l.at[i], to + i * 1024);
        if (BOTH) lds_copy16(plane2 + at + l2.at[i], to2 + i * 1024);
    }
}
// K and V of 16 keys.
template <int DP>
__device__ __forceinline__ void copy_both(const Params& a, const Source& s, const Lanes<DP>& lk, const Lanes<DP>& lv, int first,
                                          const int* ids, uint32_t k_to, uint32_t v_to) {
    if (in_one_page(a, s, first)) {
        const uint64_t row = row_of(a, s, first, ids[0]);
        copy_rows<DP>(s.k + row, lk, k_to);
        copy_rows<DP>(s.v + row, lv, v_to);
    } else {
        copy_rows_apart<DP, true>(a, s, s.k, lk, k_to, s.v, lv, v_to, first, ids);
    }
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
template <bool BF16>
__device__ __forceinline__ bool values_not_finite(const Params& a, const Tile& t, int head, int begin, int end) {
    bool bad = false;
    for (int key = max(begin, t.lo); key < min(end, t.hi); ++key) {
        const uint32_t page = min((uint32_t)a.tables[t.b * a.table_stride + page_index(a, key)], (uint32_t)a.num_pages - 1);
        const uint16_t* const v = reinterpret_cast<const uint16_t*>(
            reinterpret_cast<const uint8_t*>(a.v) + (uint64_t)page * a.page_bytes + (uint64_t)head * a.head_bytes +
            (uint64_t)(uint32_t)(key - page_index(a, key) * a.page_size) * a.row_bytes);
        for (int d = threadIdx.x & 63; d < a.dim; d += 64) {
            const float x = to_float<BF16>(v[d]);
            bad |= x - x != 0.f;
        }
    }
    return __any(bad);
}

// Whether rows whose output is not finite have to be computed again one by one: some
// key of [t.lo, t.hi) that not every row sees has a value that is not finite, or the first or
// the last one has, which stand in for the block's keys outside (a probability of 0, and
// 0 * inf is not inf), or the head is narrower than the kernel's (its padding repeats key
// elements against zeros).
template <bool BF16>
__device__ __forceinline__ bool must_repeat(const Params& a, const Tile& t, int head, int dp) {
    if (a.dim != dp) return true;
    const int first = t.first_pos + t.row0 / a.group, last = t.first_pos + (t.row0 + t.rows - 1) / a.group;
    if (values_not_finite<BF16>(a, t, head, min(first + 1, t.hi - 1), t.hi)) return true;
    return a.window > 0 && values_not_finite<BF16>(a, t, head, t.lo, max(last + 1 - a.window, t.lo + 1));
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
// head, for partial slot `slot`, or the whole of it (-1).  ONE: a sequence has one tile.
template <int MR, int KEYS, int UNIT, int WAVES, bool ONE>
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
                const int b = b0 + lane;
                const int mine = b < a.batch ? (sequence(a, b).n * a.group + MR - 1) / MR : 0;
                const int upto = before + wave_inclusive_scan(mine);
                const uint64_t past = __ballot(upto > rank);
                if (past != 0) {
                    const int l = __builtin_ctzll(past);
                    set_tile(a, b0 + l, __builtin_amdgcn_readlane(upto, l) - 1 - rank);
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
            t.b = b;
            t.q0 = __builtin_amdgcn_readlane(my.q0, b);
            t.first_pos = __builtin_amdgcn_readlane(my.first_pos, b);
            t.len = __builtin_amdgcn_readlane(my.len, b);
            t.row0 = 0;
            t.rows = __builtin_amdgcn_readlane(my.rows, b);
            t.lo = __builtin_amdgcn_readlane(my.lo, b);
            t.hi = __builtin_amdgcn_readlane(my.hi, b);
            t.base = __builtin_amdgcn_readlane(my.base, b);
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

// ---- few rows --------------------------------------------------------------------

// Up to 16 MT query rows, bound by reading the keys: 16 sequences of 2 to 32 thousand
// keys, 8 heads of 128, 754 MB, take 140 us and 6 for the join (5.2 TB/s; a copy of 4 GiB
// reads and writes 4.7).  Each wave takes blocks of 32 keys of its own, through a ring of
// two stages of its own (no barrier), and the waves' outputs meet in LDS at the end of a
// piece.  Four waves and their rings fill a CU's LDS; 64 KB are under way in it, three
// times what the memory's latency asks for at that rate.
constexpr int kFewKeys = 32;
template <int DP>
constexpr int kFewWaves = DP == 256 ? 2 : 4;
template <int DP>
constexpr int kFewUnit = kFewKeys * kFewWaves<DP>;
template <int DP>
constexpr int kFewStage = 2 * kFewKeys * DP * 2;  // K and V of a block, bytes
template <int DP>
constexpr int kFewRing = 2 * kFewStage<DP> + 4 * 256;  // a wave's: two stages, four sets of page ids

template <int DP, int MT>
constexpr int few_stage_bytes() {
    const int ring = kFewWaves<DP> * kFewRing<DP>, join = kFewWaves<DP> * 16 * MT * (DP + 4) * 4;
    return ring > join ? ring : join;
}

template <bool BF16, int DP, int MT, bool CAP>
__global__ __launch_bounds__(kFewWaves<DP> * 64) void few_rows_kernel(const Params a) {
    constexpr int WAVES = kFewWaves<DP>, MR = 16 * MT, UNIT = kFewUnit<DP>;
    constexpr int KS = DP / 32;       // steps of 32 head elements
    constexpr int DT = DP / 16;       // tiles of 16 output elements
    constexpr int kCopies = 2 * kFewKeys * DP * 2 / 1024 + 1;  // of a batch: a block, and the ids of the next but one
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    Plan& plan = *reinterpret_cast<Plan*>(smem + few_stage_bytes<DP, MT>());
    uint8_t* const ring = smem + wave * kFewRing<DP>;
    int* const ids = reinterpret_cast<int*>(ring + 2 * kFewStage<DP>);
    const auto lanes_k = lanes_of<DP>(a, k_swizzle<DP>), lanes_v = lanes_of<DP>(a, v_swizzle<DP, false>);
    const float k = unit<CAP>(a);

    Pieces<MR, kFewKeys, UNIT, WAVES, true> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        const Tile& t = piece.t;
        const int head = piece.head, u0 = piece.u0, u1 = piece.u1, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const int begin = t.base + u0 * UNIT, end = min(t.hi, t.base + u1 * UNIT);
        const int blocks = end > begin ? (end - begin + kFewKeys - 1) / kFewKeys : 0;
        const int mine = (blocks - wave + WAVES - 1) / WAVES;  // blocks wave, wave + WAVES, ...
        auto first_of = [&](int i) { return begin + (wave + i * WAVES) * kFewKeys; };
        if (mine > 0) {
            copy_pages(a, src, first_of(0) + lane, lds_addr(ids));
            copy_pages(a, src, first_of(1) + lane, lds_addr(ids + 64));
        }
        u32x4 q[MT][KS];
        int row_lo[MT], row_hi[MT];  // keys that the lane's row sees
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            load_query<KS>(a, t, head, mt * 16 + c, g, 4, q[mt]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int pos = t.first_pos + (t.row0 + mt * 16 + c) / a.group;
            row_hi[mt] = min(pos + 1, t.hi);
            row_lo[mt] = a.window > 0 ? pos + 1 - a.window : 0;
#pragma unroll
            for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(q[mt][st]));  // here, not waited for in the loop
        }
        // blocks inside [all_lo, all_hi) are seen by every row of the tile
        const int all_hi = min(t.first_pos + t.row0 / a.group + 1, t.hi);
        const int all_lo = a.window > 0 ? t.first_pos + (t.row0 + t.rows - 1) / a.group + 1 - a.window : 0;
        f32x4 o[MT][DT];
        float m[MT], z[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt] = -kInf;
            z[mt] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        auto issue = [&](int i) {  // batch i: block i, and the page ids of block i + 2
            const uint32_t st = lds_addr(ring) + (i & 1) * kFewStage<DP>;
#pragma unroll
            for (int r = 0; r < kFewKeys; r += 16) {
                copy_both<DP>(a, src, lanes_k, lanes_v, first_of(i) + r, ids + (i & 3) * 64 + r, st + r * DP * 2,
                              st + kFewStage<DP> / 2 + r * DP * 2);
            }
            copy_pages(a, src, first_of(i + 2) + lane, lds_addr(ids + ((i + 2) & 3) * 64));
        };
        if (mine > 0) {
            wait_copies<0>();
            issue(0);
            if (mine > 1) issue(1);
        }
        for (int i = 0; i < mine; ++i) {
            if (i + 1 < mine) {
                wait_copies<kCopies>();
            } else {
                wait_copies<0>();
            }
            const uint8_t* const ks = ring + (i & 1) * kFewStage<DP>;
            const uint8_t* const vs = ks + kFewStage<DP> / 2;
            const int key0 = first_of(i);
            f32x4 s[MT][2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
                const int r = kt * 16 + c;
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    const u32x4 kf = *reinterpret_cast<const u32x4*>(
                        ks + r * DP * 2 + (((4 * st + g) ^ k_swizzle<DP>(r)) * 16));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) s[mt][kt] = mfma16x16x32<BF16>(kf, q[mt][st], s[mt][kt]);
                }
            }
            const bool masked = key0 < all_lo || key0 + kFewKeys > all_hi;
            u32x4 p[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float x[8], top = -kInf;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[mt][e / 4][e % 4];
                cap_scores<CAP, 8>(a, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + (e / 4) * 16 + 4 * g + e % 4;
                    x[e] = masked & ((key < row_lo[mt]) | (key >= row_hi[mt])) ? -kInf : x[e];
                    top = fmaxf(top, x[e]);
                }
                top = max_halves(max_quarters(top));
                const float m_new = fmaxf(m[mt], top);
                if (__any((m_new - m[mt]) * k > kSlack)) {
                    const float scale = __builtin_amdgcn_exp2f((m[mt] - (m_new == -kInf ? 0.f : m_new)) * k);
                    z[mt] *= scale;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[mt][d] *= scale;
                    m[mt] = m_new;
                }
                const float shift = m[mt] == -kInf ? -kLift<BF16> : shift_of<BF16>(m[mt], k);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(x[e] * k - shift);
                    z[mt] += x[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) p[mt][e] = pack2<BF16>(x[2 * e], x[2 * e + 1]);
            }
            // O^T += V^T P^T: step slot 8 g + j is key 4 g + j (j < 4) or 16 + 4 g + j - 4
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4 vf;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const int r = kt * 16 + 4 * g + c / 4, unit = 2 * d + (c % 4) / 2;
                    const u32x2 h = read_transposed(vs + r * DP * 2 + ((unit ^ v_swizzle<DP, false>(r)) * 16) + (c & 1) * 8);
                    vf[2 * kt] = h[0];
                    vf[2 * kt + 1] = h[1];
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) o[mt][d] = mfma16x16x32<BF16>(vf, p[mt], o[mt][d]);
            }
            // the stage's reads are done (the products have taken them) before it is filled again
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (i + 2 < mine) issue(i + 2);
        }
        __syncthreads();  // every wave is done with its ring
        // ---- join the waves: rows of dim + 4 floats (maximum, sum behind the outputs)
        constexpr int kRow = DP + 4;
        float* const join = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float* const row = join + (wave * MR + mt * 16 + c) * kRow;
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(row + d * 16 + 4 * g) = o[mt][d];
            const float all = sum_halves(sum_quarters(z[mt]));
            if (g == 0) {
                row[DP] = held_max<BF16>(m[mt], k);
                row[DP + 1] = all;
            }
        }
        __syncthreads();
        bool bad = false;
        for (int row = wave; row < t.rows; row += WAVES) {
            float m2 = -kInf, sum = 0.f, w[WAVES];
#pragma unroll
            for (int v = 0; v < WAVES; ++v) m2 = fmaxf(m2, join[(v * MR + row) * kRow + DP]);
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const float mv = join[(v * MR + row) * kRow + DP];
                w[v] = mv == -kInf ? 0.f : __builtin_amdgcn_exp2f(mv - m2);
                sum += w[v] * join[(v * MR + row) * kRow + DP + 1];
            }
            const float inv = slot >= 0 ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
            uint16_t* const to = slot >= 0 ? nullptr : out_row(a, t, head, row);
            for (int d = lane; d < a.dim; d += 64) {
                float x = 0.f;
#pragma unroll
                for (int v = 0; v < WAVES; ++v) {
                    if (w[v] != 0.f) x += w[v] * join[(v * MR + row) * kRow + d];
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
        if (__any(bad) && must_repeat<BF16>(a, t, head, DP)) {
            for (int row = wave; row < t.rows; row += WAVES) {
                const int r = t.row0 + row, i = r / a.group, pos = t.first_pos + i;
                const int from = max(begin, a.window > 0 ? pos + 1 - a.window : 0), to = min(end, pos + 1);
                const RowResult x = plain_row<BF16, CAP>(a, t.b, t.q0 + i, head * a.group + r - i * a.group, max(from, 0), to);
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
        __syncthreads();  // the ring is used again
    }
    clear_rest(a);
}

// ---- many rows --------------------------------------------------------------------

// Four waves of 32 query rows each over blocks of 64 keys that they share in LDS,
// two stages: block i + 1 is copied while block i is worked on.  For calls with too few
// tiles of 256 rows to fill the chip, and heads wider than 128; two workgroups to a CU
// (one prompt of 8192 tokens, 32 heads of 128: 535 to 566 us on two cards, where 256-row
// tiles take 510 and 544).  Tiles too few to give a SIMD its second wave leave it bound by
// latency: chunks of 707 and 101 tokens, 14 heads of 64, a window of 1024 and a cap take
// 49.5 us, the vector units busy 28% of it, 0.6 waves on a SIMD.
constexpr int kManyKeys = 64, kManyWaves = 4, kManyRows = 32 * kManyWaves;
constexpr int kAhead = 4;  // operands read ahead of their products
template <int DP>
constexpr int kManyStage = 2 * kManyKeys * DP * 2;
template <int DP>
constexpr int many_stage_bytes() { return 2 * kManyStage<DP> + kManyWaves * 2 * 256; }

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
        mine.lo = a.window > 0 ? max(0, pos0 + 1 - a.window) : 0;
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
template <bool BF16, int DP, int MR, bool CAP>
__device__ __forceinline__ void store_rows(const Params& a, const Tile& t, const WaveRows<kManyKeys>& r, int wave, int head,
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
    if (__any(in && bad) && must_repeat<BF16>(a, met, head, DP)) {
        const float lift = __builtin_amdgcn_exp2f(kLift<BF16>);
        for (int row = 0; row < r.mine.rows; ++row) {
            const int at_row = r.mine.row0 + row, i = at_row / a.group, at = t.first_pos + i;
            const int from = max(begin, a.window > 0 ? at + 1 - a.window : 0);
            const RowResult x = plain_row<BF16, CAP>(a, t.b, t.q0 + i, head * a.group + at_row - i * a.group, from, min(end, at + 1));
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

template <bool BF16, int DP, bool CAP>
__global__ __launch_bounds__(kManyWaves * 64) __attribute__((amdgpu_waves_per_eu(DP == 256 ? 1 : 2)))
void many_rows_kernel(const Params a) {
    constexpr int WAVES = kManyWaves, MR = kManyRows, KEYS = kManyKeys;
    constexpr int KS = DP / 16;      // steps of 16 head elements
    constexpr int DT = DP / 32;      // tiles of 32 output elements
    constexpr int COPY = KEYS / WAVES;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    Plan& plan = *reinterpret_cast<Plan*>(smem + many_stage_bytes<DP>());
    int* const ids = reinterpret_cast<int*>(smem + 2 * kManyStage<DP>) + wave * 128;
    const auto lanes_k = lanes_of<DP>(a, k_swizzle<DP>), lanes_v = lanes_of<DP>(a, v_swizzle<DP, true>);
    const float k = unit<CAP>(a);
    // LDS places of the lane's operands in a stage: K's unit 2 st + h of row c lies st << 5 (in
    // bits 5 up) away by XOR; V's 4 rows from 4 h on, at columns of tile d, d << 6 away
    const uint32_t k_at = (uint32_t)(c * DP * 2 + ((h ^ k_swizzle<DP>(c)) * 16));
    const int vr = 4 * h + ((c & 15) >> 2);
    const uint32_t v_at = (uint32_t)(kManyStage<DP> / 2 + vr * DP * 2 +
                                     ((((c >> 4) * 2 + ((c & 3) >> 1)) ^ v_swizzle<DP, true>(vr)) * 16) + (c & 1) * 8);
    Pieces<MR, KEYS, KEYS, WAVES, false> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        const Tile& t = piece.t;
        const int head = piece.head, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const int begin = t.base + piece.u0 * KEYS, end = min(t.hi, t.base + piece.u1 * KEYS);
        const int blocks = end > begin ? (end - begin + KEYS - 1) / KEYS : 0;
        const WaveRows<KEYS> r(a, t, wave);
        u32x4 q[KS];
        load_query<KS>(a, r.mine, head, c, h, 2, q);
#pragma unroll
        for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(q[st]));  // here, not waited for in the loop
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
        float m = -kInf, z = 0.f;
        // page ids come for four blocks of the wave's 16 keys at a time, two sets in LDS
        auto pages = [&](int set) {
            copy_pages(a, src, begin + (set * 4 + (lane >> 4)) * KEYS + wave * COPY + (lane & 15), lds_addr(ids + (set & 1) * 64));
        };
        auto issue = [&](int i) {  // the wave's rows of block i
            const uint32_t st = lds_addr(smem) + (i & 1) * kManyStage<DP> + wave * COPY * DP * 2;
            copy_both<DP>(a, src, lanes_k, lanes_v, begin + i * KEYS + wave * COPY, ids + (i & 7) * 16, st,
                          st + kManyStage<DP> / 2);
            if ((i & 3) == 0 && i > 0) pages(i / 4 + 1);  // into the place of set i / 4 - 1, which is done with
        };
        if (blocks > 0) {
            pages(0);
            pages(1);
            wait_copies<0>();
            issue(0);
        }
        for (int i = 0; i < blocks; ++i) {
            // block i is there, and every wave is done with block i - 1 (in one statement: no
            // LDS read may move in between)
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (i + 1 < blocks) issue(i + 1);
            const int key0 = begin + i * KEYS;
            if (!r.sees(key0)) continue;
            const uint8_t* const st_at = smem + (i & 1) * kManyStage<DP>;
            f32x16 s[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kt][e] = 0.f;
            // products n = (st, kt) in turn, each with the read of an operand kAhead products on behind it
            auto read_k = [&](int n) {
                return *reinterpret_cast<const u32x4*>(st_at + (k_at ^ ((n / 2) << 5)) + (n % 2) * 32 * DP * 2);
            };
            u32x4 kf[kAhead];
#pragma unroll
            for (int n = 0; n < kAhead; ++n) kf[n] = read_k(n);
#pragma unroll
            for (int n = 0; n < 2 * KS; ++n) {
                __builtin_amdgcn_sched_barrier(0);
                s[n % 2] = mfma32x32x16<BF16>(kf[n % kAhead], q[n / 2], s[n % 2]);
                if (n + kAhead < 2 * KS) kf[n % kAhead] = read_k(n + kAhead);
            }
            cap_scores<CAP, 16>(a, s[0]);
            cap_scores<CAP, 16>(a, s[1]);
            r.mask(key0, h, s);
            float top = -kInf;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[kt][e]);
            top = max_halves(top);
            const float m_new = fmaxf(m, top);
            if (__any((m_new - m) * k > kSlack)) {
                const float scale = __builtin_amdgcn_exp2f((m - (m_new == -kInf ? 0.f : m_new)) * k);
                z *= scale;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= scale;
                m = m_new;
            }
            const float shift = m == -kInf ? -kLift<BF16> : shift_of<BF16>(m, k);
            // Step st of 16 keys: slot 8 h + j is key 16 st + 4 h + j (j < 4) or 16 st + 8 + 4 h + j - 4.
            // Products n = (st, d) in turn, each with the read of an operand kAhead products on and a
            // share of the next step's probabilities behind it.
            float x[8];
            auto probability = [&](int st, int e) {
                x[e] = __builtin_amdgcn_exp2f(s[st / 2][(st % 2) * 8 + e] * k - shift);
                z += x[e];
            };
            auto read_v = [&](int n) {
                const uint8_t* const at = st_at + (v_at ^ ((n % DT) << 6)) + (n / DT) * 16 * DP * 2;
                const u32x2 y0 = read_transposed(at), y1 = read_transposed(at + 8 * DP * 2);
                return u32x4{y0[0], y0[1], y1[0], y1[1]};
            };
            u32x4 vf[kAhead], p;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) vf[n] = read_v(n);
#pragma unroll
            for (int e = 0; e < 8; ++e) probability(0, e);
#pragma unroll
            for (int n = 0; n < 4 * DT; ++n) {
                const int st = n / DT, d = n % DT;
                if (d == 0) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = pack2<BF16>(x[2 * e], x[2 * e + 1]);
                }
                __builtin_amdgcn_sched_barrier(0);
                o[d] = mfma32x32x16<BF16>(vf[n % kAhead], p, o[d]);
                if (n + kAhead < 4 * DT) vf[n % kAhead] = read_v(n + kAhead);
                if (st < 3) {
#pragma unroll
                    for (int e = d * 8 / DT; e < (d + 1) * 8 / DT; ++e) probability(st + 1, e);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        store_rows<BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held_max<BF16>(m, k), z, o);
        __syncthreads();  // every wave is done with the stages
    }
    clear_rest(a);
}

// ---- a great many rows -----------------------------------------------------------------

// Eight waves of 32 rows, two on each SIMD, that take turns: while waves 0 to 3 are in
// their products (scores of block i + 1, outputs of block i), waves 4 to 7 make the
// probabilities of a block, and the other way round.  Both phases take about as long, so
// the matrix cores and the vector units are busy together; the same work in any order of
// the waves' own left each idle half of the time (two four-wave workgroups a CU: 4% slower
// on a prompt of 8192 tokens, 32 heads of 128).  Waves 0 to 3 copy K, waves 4 to 7 copy V,
// three blocks of each in LDS.  510 to 544 us by the card, 1010 to 1078 TFLOP/s, where the
// library's large matrix product reaches 1184 on the fastest; by the counters the matrix
// cores are busy 50% of the cycles and vector instructions take 49%.
constexpr int kWideWaves = 8, kWideRows = 32 * kWideWaves, kWideRing = 3;
template <int DP>
constexpr int kWideBlock = kManyKeys * DP * 2;  // bytes of K, or of V
template <int DP>
constexpr int wide_stage_bytes() { return 2 * kWideRing * kWideBlock<DP> + kWideWaves * 2 * 256; }

template <bool BF16, int DP, bool CAP>
__global__ __launch_bounds__(kWideWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void wide_rows_kernel(const Params a) {
    constexpr int MR = kWideRows, KEYS = kManyKeys, KS = DP / 16, DT = DP / 32;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    Plan& plan = *reinterpret_cast<Plan*>(smem + wide_stage_bytes<DP>());
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    const bool late = wave >= 4;  // half a turn behind, and copies V
    int* const ids = reinterpret_cast<int*>(smem + 2 * kWideRing * kWideBlock<DP>) + wave * 128;
    const uint32_t my_ring = lds_addr(smem) + (late ? kWideRing * kWideBlock<DP> : 0) + (wave & 3) * 16 * DP * 2;
    const auto lanes = lanes_of<DP>(a, [&](int row) { return late ? v_swizzle<DP, true>(row) : k_swizzle<DP>(row); });
    const float k = unit<CAP>(a);
    const uint32_t k_at = (uint32_t)(c * DP * 2 + ((h ^ k_swizzle<DP>(c)) * 16));
    const int vr = 4 * h + ((c & 15) >> 2);
    const uint32_t v_at = (uint32_t)(vr * DP * 2 + ((((c >> 4) * 2 + ((c & 3) >> 1)) ^ v_swizzle<DP, true>(vr)) * 16) +
                                     (c & 1) * 8);
    Pieces<MR, KEYS, KEYS, kWideWaves, false> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        const Tile& t = piece.t;
        const int head = piece.head, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const int begin = t.base + piece.u0 * KEYS, end = min(t.hi, t.base + piece.u1 * KEYS);
        const int blocks = end > begin ? (end - begin + KEYS - 1) / KEYS : 0;
        const WaveRows<KEYS> r(a, t, wave);
        const uint8_t* const plane = late ? src.v : src.k;
        const int mine0 = begin + (wave & 3) * 16;  // of block 0, the first key that the wave copies
        // page ids come for four blocks of the wave's 16 keys at a time, two sets in LDS
        auto pages = [&](int set) {
            copy_pages(a, src, mine0 + (set * 4 + (lane >> 4)) * KEYS + (lane & 15), lds_addr(ids + (set & 1) * 64));
        };
        auto copy = [&](int j, int place, int id) {  // the wave's keys of block j, `id` the first one's page
            const int first = mine0 + j * KEYS;
            const uint32_t to = my_ring + place * kWideBlock<DP>;
            if (__builtin_expect(in_one_page(a, src, first), 1)) {
                copy_rows<DP>(plane + row_of(a, src, first, id), lanes, to);
            } else {
                copy_rows_apart<DP, false>(a, src, plane, lanes, to, plane, lanes, to, first, ids + (j & 7) * 16);
            }
        };
        if (blocks > 0) {
            pages(0);
            pages(1);
        }
        u32x4 q[KS];
        load_query<KS>(a, r.mine, head, c, h, 2, q);
#pragma unroll
        for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(q[st]));  // here, not waited for in the loop
        f32x16 o[DT], s[2];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
        u32x4 p[4];
        float m = -kInf, z = 0.f;
        if (blocks > 0) {
            wait_copies<0>();
            copy(0, 0, ids[0]);
            if (blocks > 1) copy(1, 1, ids[16]);
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (late) asm volatile("s_barrier" ::: "memory");
            // (The expectations lay the usual way through a turn out without branches: the prompt
            // of 8192 tokens 532 us without them, 528 with.)
            int place = 2;  // ring place of block i + 3
            for (int i = -1; i < blocks; ++i) {
                // ---- products: scores of block i + 1, outputs of block i
                const int next = begin + (i + 1) * KEYS;
                const int place_next = place == 2 ? 0 : place + 1;  // of blocks i + 1 (and i + 4)
                const int place_now = place;                        // of blocks i (and i + 3)
                const bool do_next = i + 1 < blocks && r.sees(next), do_now = i >= 0 && r.sees(next - KEYS);
                const int id = ids[((i + 3) & 7) * 16];
                __builtin_amdgcn_s_setprio(1);
                if (__builtin_expect(do_next, 1)) {
                    const uint8_t* const st_at = smem + place_next * kWideBlock<DP>;
                    auto read_k = [&](int n) {
                        return *reinterpret_cast<const u32x4*>(st_at + (k_at ^ ((n / 2) << 5)) + (n % 2) * 32 * DP * 2);
                    };
                    u32x4 kf[kAhead];
#pragma unroll
                    for (int n = 0; n < kAhead; ++n) kf[n] = read_k(n);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[kt][e] = 0.f;
#pragma unroll
                    for (int n = 0; n < 2 * KS; ++n) {
                        __builtin_amdgcn_sched_barrier(0);
                        s[n % 2] = mfma32x32x16<BF16>(kf[n % kAhead], q[n / 2], s[n % 2]);
                        if (n + kAhead < 2 * KS) kf[n % kAhead] = read_k(n + kAhead);
                    }
                }
                if (__builtin_expect(do_now, 1)) {
                    const uint8_t* const st_at = smem + (kWideRing + place_now) * kWideBlock<DP>;
                    auto read_v = [&](int n) {
                        const uint8_t* const at = st_at + (v_at ^ ((n % DT) << 6)) + (n / DT) * 16 * DP * 2;
                        const u32x2 y0 = read_transposed(at), y1 = read_transposed(at + 8 * DP * 2);
                        return u32x4{y0[0], y0[1], y1[0], y1[1]};
                    };
                    u32x4 vf[kAhead];
#pragma unroll
                    for (int n = 0; n < kAhead; ++n) vf[n] = read_v(n);
#pragma unroll
                    for (int n = 0; n < 4 * DT; ++n) {
                        __builtin_amdgcn_sched_barrier(0);
                        o[n % DT] = mfma32x32x16<BF16>(vf[n % kAhead], p[n / DT], o[n % DT]);
                        if (n + kAhead < 4 * DT) vf[n % kAhead] = read_v(n + kAhead);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                // ---- probabilities of block i + 1; copies of block i + 3
                if (i + 3 < blocks) {
                    if (((i + 3) & 3) == 0) pages((i + 3) / 4 + 1);  // into the place of the set before, which is done with
                    copy(i + 3, place_now, id);
                }
                if (__builtin_expect(do_next, 1)) {
                    cap_scores<CAP, 16>(a, s[0]);
                    cap_scores<CAP, 16>(a, s[1]);
                    r.mask(next, h, s);
                    float top = -kInf;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[kt][e]);
                    top = max_halves(top);
                    const float m_new = fmaxf(m, top);
                    if (__builtin_expect(__any((m_new - m) * k > kSlack), 0)) {
                        const float scale = __builtin_amdgcn_exp2f((m - (m_new == -kInf ? 0.f : m_new)) * k);
                        z *= scale;
#pragma unroll
                        for (int d = 0; d < DT; ++d) o[d] *= scale;
                        m = m_new;
                    }
                    const float shift = m == -kInf ? -kLift<BF16> : shift_of<BF16>(m, k);
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            x[e] = __builtin_amdgcn_exp2f(s[st / 2][(st % 2) * 8 + e] * k - shift);
                            z += x[e];
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[st][e] = pack2<BF16>(x[2 * e], x[2 * e + 1]);
                    }
                }
                // the last turn's copies have landed; this turn's may be under way
                if (i + 3 < blocks) {
                    wait_copies<Lanes<DP>::kSteps>();
                } else {
                    wait_copies<0>();
                }
                asm volatile("s_barrier" ::: "memory");
                place = place_next;
            }
            if (!late) asm volatile("s_barrier" ::: "memory");
        }
        store_rows<BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held_max<BF16>(m, k), z, o);
        __syncthreads();  // every wave is done with the ring
    }
    clear_rest(a);
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

// ---- host ----------------------------------------------------------------------------

struct Call {
    Params p;
    int dp, tile_rows, grid;   // tile_rows: 16 or 32 (few rows), 128 or 256
    int64_t tiles;             // at most
    size_t bytes;
};

int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Which kernel, tiles and split, from what the host knows.  `a` has passed check().
Call plan_call(const pw4_paged_attention_args* a) {
    Call c{};
    Params& p = c.p;
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
    p.page_bytes = (uint32_t)a->page_stride * 2;
    p.row_bytes = (uint32_t)a->row_stride * 2;
    p.head_bytes = (uint32_t)a->kv_head_stride * 2;
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
    p.flat = (uint64_t)a->page_size * p.row_bytes > UINT32_MAX ? 0 : p.page_shift >= 4 ? 2 : a->page_size % 8 == 0 ? 1 : 0;
    p.cap2 = a->softcap > 0.f ? cap * kLog2e : 0.f;
    const int64_t rows = (int64_t)p.max_q * p.group;
    c.dp = padded_dim(a->head_dim);
    const int cus = device_cus();
    const auto tiles_of = [&](int tile_rows) {
        return std::min(a->num_tokens * p.group / tile_rows + p.batch, p.batch * ceil_div(rows, tile_rows));
    };
    // 256-row tiles run at the higher rate, but only one to a CU
    c.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32
                  : c.dp == 256 || tiles_of(kWideRows) * p.kv_heads < cus ? kManyRows : kWideRows;
    if (const char* const forced = plan_override("PW4_ATTN_TILE"); forced && c.tile_rows > 32 && c.dp != 256) {
        c.tile_rows = forced[0] == '2' ? kWideRows : kManyRows;
    }
    const bool few = c.tile_rows <= 32;
    c.tiles = few ? p.batch : tiles_of(c.tile_rows);
    const int unit = !few ? kManyKeys : c.dp == 64 ? kFewUnit<64> : c.dp == 128 ? kFewUnit<128> : kFewUnit<256>;
    // workgroups that run at once
    const int slots = few ? (c.dp == 64 ? 2 * cus : cus) : c.tile_rows == kManyRows && c.dp != 256 ? 2 * cus : cus;
    // Units of a tile: of the keys that a window leaves its rows, or all.  (Its first block may begin
    // early.)  32 query on 8 key-value heads of 128, sequences of 32768 keys, the rules below by
    // these units and by all of the sequence's, us: 8 tokens in a window of 128 7.1 and 9.7, two
    // chunks of 100 in one of 512 22.6 and 45.1, in one of 128 15.4 and 49.0.
    const int64_t most_keys =
        p.window == 0 ? p.max_len
                      : std::min<int64_t>(p.max_len, (int64_t)p.window + (std::min<int64_t>(c.tile_rows, rows) + p.group - 2) / p.group);
    const int64_t most_units = ceil_div(most_keys, unit) + 1;
    const char* const forced = plan_override("PW4_ATTN_UNITS");
    const int forced_units = forced ? std::atoi(forced) : 0;
    // A few rows: whole, a workgroup takes about 1.1 us a unit of 128 keys; the split, a second
    // launch and the partial outputs' way through memory, which grow with the tiles.  8 key-value
    // heads, sequences of one length, whole and split, us:
    //   heads of 64   1 of 640 keys 9.2 and 10.9, of 777 11.1 and 10.8, of 8000 60 and 20
    //                 8 of 1600 16.6 and 17.5, of 2400 22.4 and 20.5; 16 of 2400 22.6 and 25.2, of 4000 33.9 and 32.3
    //   heads of 128  1 of 640 11.2 and 12.4, of 777 13.7 and 12.3, of 8000 72 and 22; 4 of 1100 16.2 and 19.0
    //                 8 of 1600 21.3 and 22.3, of 2400 27.6 and 26.1; 16 of 2400 29.8 and 35.2, of 4000 43.8 and 48.1
    //   heads of 256 (units of 64 keys)  1 of 400 20.5 and 15.1; 8 of 777 32.4 and 28.8, of 1100 40.9 and 31.4
    //                 16 of 1100 41.6 and 37.5, of 1600 52.7 and 48.2
    // Over 1 to 16 sequences of 400 to 8000 keys the thresholds' choice is within 17% of the better
    // one, for each of these heads.  Lengths of one batch that differ are not looked at,
    // max_seq_len is.
    // Else where the tiles leave at least half of the chip idle and are long, since a piece's
    // partial outputs are written and read again: 270 tiles of 128 rows on 512 places, 18 blocks
    // each, take 49.5 us whole and 63 split.  The rule still splits some calls that are faster
    // whole: two chunks of 100 tokens in a window of 1024 take 32.0 us whole and 35.9 split.
    p.min_units = forced_units > 0 ? forced_units : few ? 1 : 8;
    const char* const forced_split = plan_override("PW4_ATTN_SPLIT");
    const bool wanted = forced_split ? forced_split[0] == '1'
                        : few ? most_units > (8 * c.tiles * p.kv_heads <= cus ? 7 : 4 * c.tiles * p.kv_heads <= cus ? 16 : 22)
                              : 2 * c.tiles * p.kv_heads <= slots && most_units > 2 * p.min_units;
    p.split = wanted && c.tiles > 0 && p.batch <= kMaxSplitTiles && c.tiles <= kMaxSplitTiles && c.tiles * p.kv_heads * most_units < INT_MAX;
    c.grid = (int)(c.tiles * p.kv_heads);
    if (p.split) {
        c.grid = (int)std::min<int64_t>(slots, ceil_div(c.tiles * p.kv_heads * most_units, p.min_units));
        const int64_t rows_held = 2 * (int64_t)c.grid * c.tile_rows;
        c.bytes = (size_t)(rows_held * (p.dim + 2) + PlanOut::kInts) * 4;
    }
    return c;
}

// Runs a kernel with more LDS than a kernel may have unasked; the permission is
// asked for once a kernel and device.
template <auto Kernel>
hipError_t run(const Call& c, int waves, int stages, hipStream_t s) {
    const int most = stages + (int)sizeof(Plan), lds = c.p.split ? most : stages;
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
    if (dev < 0 || dev >= 64 || (allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != hipSuccess) return e;
        if (dev >= 0 && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(Kernel, dim3((unsigned)std::max(c.grid, 1)), dim3(waves * 64), lds, s, c.p);
    return hipGetLastError();
}

template <bool BF16, int DP, bool CAP>
hipError_t launch(const Call& c, hipStream_t s) {
    hipError_t e;
    if (c.tile_rows == 16) {
        e = run<few_rows_kernel<BF16, DP, 1, CAP>>(c, kFewWaves<DP>, few_stage_bytes<DP, 1>(), s);
    } else if (c.tile_rows == 32) {
        e = run<few_rows_kernel<BF16, DP, 2, CAP>>(c, kFewWaves<DP>, few_stage_bytes<DP, 2>(), s);
    } else if (c.tile_rows == kManyRows) {
        e = run<many_rows_kernel<BF16, DP, CAP>>(c, kManyWaves, many_stage_bytes<DP>(), s);
    } else if constexpr (DP < 256) {
        e = run<wide_rows_kernel<BF16, DP, CAP>>(c, kWideWaves, wide_stage_bytes<DP>(), s);
    } else {
        e = hipErrorInvalidValue;  // no such tile: plan_call
    }
    if (e != hipSuccess || !c.p.split) return e;
    const dim3 grid((unsigned)(c.tiles * c.p.kv_heads), c.tile_rows / 4);
    if (c.tile_rows == 16) {
        hipLaunchKernelGGL((join_kernel<16, BF16>), grid, dim3(256), 0, s, c.p, c.grid);
    } else if (c.tile_rows == 32) {
        hipLaunchKernelGGL((join_kernel<32, BF16>), grid, dim3(256), 0, s, c.p, c.grid);
    } else if (c.tile_rows == kManyRows) {
        hipLaunchKernelGGL((join_kernel<kManyRows, BF16>), grid, dim3(256), 0, s, c.p, c.grid);
    } else {
        hipLaunchKernelGGL((join_kernel<kWideRows, BF16>), grid, dim3(256), 0, s, c.p, c.grid);
    }
    return hipGetLastError();
}

template <bool BF16, int DP>
hipError_t launch_cap(const Call& c, hipStream_t s) {
    return c.p.cap2 > 0.f ? launch<BF16, DP, true>(c, s) : launch<BF16, DP, false>(c, s);
}
template <bool BF16>
hipError_t launch_dim(const Call& c, hipStream_t s) {
    return c.dp == 64 ? launch_cap<BF16, 64>(c, s) : c.dp == 128 ? launch_cap<BF16, 128>(c, s) : launch_cap<BF16, 256>(c, s);
}

int check(const pw4_paged_attention_args* a) {
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
    const uint64_t addresses = (uint64_t)(uintptr_t)a->q | (uint64_t)(uintptr_t)a->k_cache |
                               (uint64_t)(uintptr_t)a->v_cache | (uint64_t)(uintptr_t)a->out;
    const uint64_t strides = (uint64_t)(a->q_token_stride | a->q_head_stride | a->page_stride | a->row_stride |
                                        a->kv_head_stride);
    if ((addresses & 15) != 0 || (strides & 7) != 0) return PW4_ERR_ARG;
    for (int64_t v : {a->page_stride, a->row_stride, a->kv_head_stride}) {
        if (v < 0) return PW4_ERR_ARG;
        if (v > INT_MAX) return PW4_ERR_SHAPE;
    }
    if (a->row_stride >= 1 << 24) return PW4_ERR_SHAPE;
    return PW4_OK;
}

}  // namespace

extern "C" {

size_t pw4_paged_attention_workspace_size(const pw4_paged_attention_args* args) {
    return check(args) != PW4_OK || args->num_tokens == 0 ? 0 : plan_call(args).bytes;
}

int pw4_paged_attention(const pw4_paged_attention_args* args, void* workspace, size_t workspace_bytes,
                        pw4_stream_t stream) {
    if (const int rc = check(args)) return rc;
    if (args->num_tokens == 0) return PW4_OK;
    Call c = plan_call(args);
    if (c.grid > 65535 * 4096 || c.tiles * c.p.kv_heads > INT_MAX) return PW4_ERR_SHAPE;
    if (c.bytes > 0) {
        if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < c.bytes) {
            return PW4_ERR_WORKSPACE;
        }
        const int64_t rows = 2 * (int64_t)c.grid * c.tile_rows;
        c.p.part_o = static_cast<float*>(workspace);
        c.p.part_ml = c.p.part_o + rows * c.p.dim;
        c.p.plan = reinterpret_cast<int32_t*>(c.p.part_ml + rows * 2);
    }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const hipError_t e = args->dtype == PW4_DTYPE_BF16 ? launch_dim<true>(c, s) : launch_dim<false>(c, s);
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // extern "C"

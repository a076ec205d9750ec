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
#include "paged_attention_parts.h"

using namespace pw4;

namespace {

// The cache's elements one at a time.
struct HalfKeys {
    static constexpr bool kRepeats = true, kFresh = false;
    template <bool BF16>
    static __device__ __forceinline__ float element(const Params& a, const uint16_t* plane, int head, uint32_t page,
                                                    uint32_t row, int d) {
        const uint64_t at = (uint64_t)page * a.page_bytes + (uint64_t)row * a.row_bytes + (uint64_t)head * a.head_bytes;
        return to_float<BF16>(reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(plane) + at)[d]);
    }
};

// ---- copying a block of keys into LDS --------------------------------------------

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
        join_waves<HalfKeys, BF16, DP, MT, WAVES, CAP>(a, t, smem, wave, head, slot, begin, end, k, m, z, o);
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
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;
constexpr int kAhead = 4;  // operands read ahead of their products
template <int DP>
constexpr int kManyStage = 2 * kManyKeys * DP * 2;
template <int DP>
constexpr int many_stage_bytes() { return 2 * kManyStage<DP> + kManyWaves * 2 * 256; }

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
        store_rows<HalfKeys, BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held_max<BF16>(m, k), z, o);
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
        store_rows<HalfKeys, BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held_max<BF16>(m, k), z, o);
        __syncthreads();  // every wave is done with the ring
    }
    clear_rest(a);
}

// ---- host ----------------------------------------------------------------------------

struct Call {
    Params p;
    int dp, tile_rows, grid;   // tile_rows: 16 or 32 (few rows), 128 or 256
    int64_t tiles;             // at most
    size_t bytes;
};

// Which kernel, tiles and split, from what the host knows.  `a` has passed check().
Call plan_call(const pw4_paged_attention_args* a) {
    Call c{};
    Params& p = c.p;
    p = params_of(a);
    p.page_bytes = (uint32_t)a->page_stride * 2;
    p.row_bytes = (uint32_t)a->row_stride * 2;
    p.head_bytes = (uint32_t)a->kv_head_stride * 2;
    p.flat = (uint64_t)a->page_size * p.row_bytes > UINT32_MAX ? 0 : p.page_shift >= 4 ? 2 : a->page_size % 8 == 0 ? 1 : 0;
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
        c.bytes = partial_bytes(c.grid, c.tile_rows, p.dim);
    }
    return c;
}

template <bool BF16, int DP, bool CAP>
hipError_t launch(const Call& c, hipStream_t s) {
    hipError_t e;
    if (c.tile_rows == 16) {
        e = run_attention<few_rows_kernel<BF16, DP, 1, CAP>>(c.p, c.grid, kFewWaves<DP>, few_stage_bytes<DP, 1>(), c.p.split ? (int)sizeof(Plan) : 0, s);
    } else if (c.tile_rows == 32) {
        e = run_attention<few_rows_kernel<BF16, DP, 2, CAP>>(c.p, c.grid, kFewWaves<DP>, few_stage_bytes<DP, 2>(), c.p.split ? (int)sizeof(Plan) : 0, s);
    } else if (c.tile_rows == kManyRows) {
        e = run_attention<many_rows_kernel<BF16, DP, CAP>>(c.p, c.grid, kManyWaves, many_stage_bytes<DP>(), c.p.split ? (int)sizeof(Plan) : 0, s);
    } else if constexpr (DP < 256) {
        e = run_attention<wide_rows_kernel<BF16, DP, CAP>>(c.p, c.grid, kWideWaves, wide_stage_bytes<DP>(), c.p.split ? (int)sizeof(Plan) : 0, s);
    } else {
        e = hipErrorInvalidValue;  // no such tile: plan_call
    }
    if (e != hipSuccess || !c.p.split) return e;
    if (c.tile_rows == 16) {
        run_join<16, BF16>(c.p, c.tiles, c.grid, s);
    } else if (c.tile_rows == 32) {
        run_join<32, BF16>(c.p, c.tiles, c.grid, s);
    } else if (c.tile_rows == kManyRows) {
        run_join<kManyRows, BF16>(c.p, c.tiles, c.grid, s);
    } else {
        run_join<kWideRows, BF16>(c.p, c.tiles, c.grid, s);
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
    if (const int rc = check_attention(a)) return rc;
    if (a->num_tokens == 0) return PW4_OK;
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
    const int waves = c.tile_rows > kManyRows ? kWideWaves : c.tile_rows > 32 ? kManyWaves
                      : c.dp == 64 ? kFewWaves<64> : c.dp == 128 ? kFewWaves<128> : kFewWaves<256>;
    if (!fits_a_launch(c.tiles * c.p.kv_heads, waves)) return PW4_ERR_SHAPE;
    if (c.bytes > 0) {
        if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < c.bytes) {
            return PW4_ERR_WORKSPACE;
        }
        place_partials(c.p, workspace, c.grid, c.tile_rows);
    }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const hipError_t e = args->dtype == PW4_DTYPE_BF16 ? launch_dim<true>(c, s) : launch_dim<false>(c, s);
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // extern "C"

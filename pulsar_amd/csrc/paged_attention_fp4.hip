// Attention of new tokens over a paged cache in 4 bits (the definition and the pages'
// layout: pulsar_paged.h).
//
// A key is codes times powers of two, one for each 32 elements.  The conversion
// instructions take both (v_cvt_scalef32_pk_*_fp4: two elements each), and every value
// that the append stores is exact in 16 bits but for fp16's subnormal ones, which are
// rounded as reading them back rounds them; so the products see the cache's own
// numbers and the rest is the attention over a 16-bit cache: rows, tiles, transposed
// products and splitting are those of paged_attention.hip.
//
// Scores, maxima and sums are fp32.  The probabilities are rounded to 16 bits, as over a 16-bit cache: the
// matrix instructions take both operands in one type, and a second product of what the rounding leaves would
// be half of their work again.  The sums are of the unrounded ones.  (Against 64 bits, relative to the
// outputs' norm: 2.0e-3 to 2.3e-3 in bf16, of which 1.5e-3 to 1.7e-3 is the outputs' own rounding, and
// 2.9e-4 and 2.1e-4 in fp16.)
//
// Keys come into registers as they lie in the cache, a block ahead; a wave's load takes 16
// keys, lane l a quarter (l / 16) of key l % 16's head.  Widened, that quarter is K's matrix
// operand as it is, q's elements being put in the same order; V goes to LDS (and K too, where
// waves share it), from where it is read transposed.  A key index outside what some row of the
// tile sees is clamped to one that is seen, as there.
//
// Three kernels, by the rows of a tile (plan_call has the rules and both sides' times); their bounds on
// an MI355X, heads of 128, 4 query heads on each of 8 key-value heads, bf16:
//   16, 32   waves with keys of their own.  Memory: 16 tokens over 2 to 32 thousand keys, 200 MB, 41 us (4.9
//            TB/s, what a copy reaches) and 5.8 for the join; vector units 42% busy.
//   128      four waves share blocks of 64 keys.  Latency, with a wave or two on a SIMD: 6 chunks of 101 and
//            707 tokens in a window of 1024 keys (heads of 64, a cap), 35 us.
//   256      eight waves in turns.  A prompt of 8192 tokens 530 to 560 us, 1.0 PFLOP/s: matrix cores 43% and
//            vector units 48% busy; over 16-bit keys 515, the rest is the widening.
#include "paged_attention_parts.h"

#include <type_traits>

using namespace pw4;

namespace {

struct Fp4Params : Params {
    uint32_t row_codes, row_exps;    // bytes of a token's codes, and of its exponents
    uint32_t head_codes, head_exps;  // of a page's of one head
    uint32_t exps_at;                // where a page's exponents begin
    uint32_t index_magic;            // key / page_size = (2 key * magic) >> (32 + shift), for any page size
    int32_t index_shift;
};

// The cache's elements one at a time, as the products take them.
struct Fp4Keys {
    static constexpr bool kRepeats = false, kFresh = true;
    template <bool BF16>
    static __device__ __forceinline__ float element(const Fp4Params& a, const uint16_t* plane, int head, uint32_t page,
                                                    uint32_t row, int d) {
        const uint8_t* const at = reinterpret_cast<const uint8_t*>(plane) + (uint64_t)page * a.page_bytes;
        const uint32_t code = at[head * a.head_codes + row * a.row_codes + d / 2] >> (d % 2 * 4) & 15;
        const uint32_t exp = at[a.exps_at + head * a.head_exps + row * a.row_exps + d / 32];
        const float scale = __builtin_bit_cast(float, exp << 23);
        const auto pair = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0);
        return to_float<BF16>(f32_to_out<BF16>(pair[0]));
    }
};

// Where a tile's keys are.
struct Source {
    const uint8_t* k;
    const uint8_t* v;
    const int32_t* table;    // the sequence's row
    uint32_t codes, exps;    // of the key-value head in a page
    uint32_t pages1;         // pages - 1
    int lo, last;            // keys are clamped to [lo, last]
};
__device__ __forceinline__ Source source_of(const Fp4Params& a, const Tile& t, int head) {
    return Source{reinterpret_cast<const uint8_t*>(a.k), reinterpret_cast<const uint8_t*>(a.v), a.tables + t.b * a.table_stride,
                  head * a.head_codes, a.exps_at + head * a.head_exps, (uint32_t)a.num_pages - 1, t.lo, t.hi - 1};
}
__device__ __forceinline__ int clamp_key(const Source& s, int key) { return min(max(key, s.lo), s.last); }

// A lane's quarter of a key, as it lies in the cache: DP / 4 elements.
template <int DP>
struct Quarter {
    static constexpr int kWords = DP / 32;            // of 8 codes
    static constexpr int kExps = DP == 256 ? 2 : 1;
    uint32_t codes[kWords], exps[kExps];
};

// Where in a token's codes and exponents a lane's quarter is.  Heads narrower than DP: a quarter, or
// half of one, that they do not have is read from the head's start, and its exponent taken as 0.
template <int DP>
struct Lane {
    uint32_t codes[Quarter<DP>::kExps], exps[Quarter<DP>::kExps];
    bool there[Quarter<DP>::kExps];
    __device__ __forceinline__ Lane(const Fp4Params& a, int g) {
#pragma unroll
        for (int h = 0; h < Quarter<DP>::kExps; ++h) {
            const int first = g * (DP / 4) + h * 32;  // element
            there[h] = first < a.dim;
            codes[h] = there[h] ? first / 2 : 0;
            exps[h] = there[h] ? first / 32 : 0;
        }
    }
};

template <int DP>
__device__ __forceinline__ void load_quarter(const uint8_t* codes, const uint8_t* exps, const Lane<DP>& l, Quarter<DP>& q) {
    if constexpr (DP == 64) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(codes + l.codes[0]);
        q.codes[0] = x[0];
        q.codes[1] = x[1];
    } else {
#pragma unroll
        for (int h = 0; h < Quarter<DP>::kExps; ++h) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(codes + l.codes[h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) q.codes[4 * h + e] = x[e];
        }
    }
#pragma unroll
    for (int h = 0; h < Quarter<DP>::kExps; ++h) q.exps[h] = exps[l.exps[h]];
}

// A lane's key of 16: its page's id, which takes a load, and its row of the page.
struct Key {
    uint32_t page, row;
};
// The lane's quarters of key c of 16 keys, in two steps: where it is, and its codes and exponents.
template <int DP>
struct Loader {
    Lane<DP> lane;
    int c;
    __device__ __forceinline__ Loader(const Fp4Params& a, int l) : lane(a, l >> 4), c(l & 15) {}
    __device__ __forceinline__ Key find(const Fp4Params& a, const Source& s, int first) const {
        const uint32_t key = clamp_key(s, first + c), index = __umulhi(2 * key, a.index_magic) >> a.index_shift;
        return Key{(uint32_t)s.table[index], key - index * (uint32_t)a.page_size};
    }
    // `plane` with the head's place in a page: codes, exponents
    __device__ __forceinline__ void load(const Fp4Params& a, const Source& s, const uint8_t* plane, const Key& key,
                                         Quarter<DP>& q) const {
        const uint8_t* const page = plane + (uint64_t)min(key.page, s.pages1) * a.page_bytes;
        load_quarter<DP>(page + (s.codes + __umul24(key.row, a.row_codes)), page + (s.exps + __umul24(key.row, a.row_exps)), lane, q);
    }
};

// 16-bit elements of a quarter: word i becomes elements 8 i .. 8 i + 7.
template <bool BF16, int DP>
__device__ __forceinline__ u32x4 widen(const Lane<DP>& l, const Quarter<DP>& q, int i) {
    const int h = DP == 256 ? i / 4 : 0;
    const float scale = __builtin_bit_cast(float, (l.there[h] ? q.exps[h] : 127u) << 23);
    const uint32_t w = q.codes[i];
    if constexpr (BF16) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
    } else {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
    }
}
// Where quarter g of row r of a stage begins, in bytes: rows of DP 16-bit elements, their 16-byte
// units placed by XOR with `swizzle`; word i is (i << 4) away by XOR.
template <int DP>
__device__ __forceinline__ uint32_t quarter_at(int g, int r, int swizzle) {
    return r * DP * 2 + ((g * Quarter<DP>::kWords) ^ swizzle) * 16;
}
// The quarter, widened.
template <bool BF16, int DP>
__device__ __forceinline__ void store_quarter(uint8_t* stage, uint32_t at, const Lane<DP>& l, const Quarter<DP>& q) {
#pragma unroll
    for (int i = 0; i < Quarter<DP>::kWords; ++i) {
        *reinterpret_cast<u32x4*>(stage + (at ^ (i << 4))) = widen<BF16, DP>(l, q, i);
    }
}

// The transposing read at LDS[at + i * STEP].
template <int STEP>
__device__ __forceinline__ u32x2 transposed(uint32_t at, int i) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    using Lds = __attribute__((address_space(3))) s16x4*;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(uintptr_t)at + i * (STEP / 8)));
}

// ---- few rows --------------------------------------------------------------------

// 16 MT query rows, of a sequence that has no more or one of its tiles.  Each wave takes blocks of 32 keys
// of its own: K straight from registers, V through 32 rows of LDS of its own (no barrier); the next block's
// codes are under way during the softmax and the second product.  Memory is hidden by waves, so registers
// are held to four a SIMD (16 rows, heads of 128; 53 us for 200 MB of keys where two had 76) and to three (32
// rows; 79 us where two had 85), for which the queries lie in LDS.
constexpr int kFewKeys = 32;
constexpr int kAhead = 4;  // operands read ahead of their products
template <int DP>
constexpr int kFewWaves = DP == 256 ? 2 : 4;
template <int DP>
constexpr int kFewUnit = kFewKeys * kFewWaves<DP>;
template <int DP>
constexpr int kFewStage = kFewKeys * DP * 2;  // V of a block, bytes

// Whether the queries lie in LDS, operand by operand, rather than in every wave's registers.
template <int DP, int MT>
constexpr bool kQueryInLds = DP == 128 && MT == 2;
template <int DP, int MT>
constexpr int few_stage_bytes() {
    const int stages = kFewWaves<DP> * kFewStage<DP> + (kQueryInLds<DP, MT> ? 16 * MT * DP * 2 : 0), join = kFewWaves<DP> * 16 * (DP + 4) * 4;  // 16 rows at a time
    return stages > join ? stages : join;
}

// Waves on a SIMD that a kernel's registers are held to.
template <int DP, int MT>
constexpr int kFewOccupancy = DP == 64 ? MT == 1 ? 5 : 3 : DP == 128 ? MT == 1 ? 4 : 3 : MT == 1 ? 2 : 1;
// Its workgroups on a CU, by these and by LDS (160 KB), with `plan` bytes behind the stages.
template <int DP, int MT>
int few_slots(int plan) {
    return std::min(kFewOccupancy<DP, MT> * 4 / kFewWaves<DP>, (160 << 10) / (few_stage_bytes<DP, MT>() + plan));
}

// ONE: a sequence has one tile; else the call is not split.
template <bool BF16, int DP, int MT, bool CAP, bool ONE>
__global__ __launch_bounds__(kFewWaves<DP> * 64) __attribute__((amdgpu_waves_per_eu(kFewOccupancy<DP, MT>)))
void fp4_few_rows_kernel(const Fp4Params a) {
    constexpr int WAVES = kFewWaves<DP>, MR = 16 * MT, UNIT = kFewUnit<DP>;
    constexpr int KS = DP / 32;       // steps of 32 head elements
    constexpr int DT = DP / 16;       // tiles of 16 output elements
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Plan& plan = *reinterpret_cast<Plan*>(smem + few_stage_bytes<DP, MT>());
    uint8_t* const stage = smem + wave * kFewStage<DP>;
    const float k = unit<CAP>(a);

    Pieces<MR, kFewKeys, UNIT, WAVES, ONE, ONE, !ONE> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        // (made anew for each piece: held through all of them, what depends on it takes registers)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int c = lane & 15, g = lane >> 4;
        const Loader<DP> from(a, lane);
        // LDS places, the second 16 rows' as the first's: the lane's quarter of V's row c; of 4 rows from 4 g on,
        // the columns of tile 0 (of tile d: d << 5 away by XOR)
        const uint32_t v_to = quarter_at<DP>(g, c, v_swizzle<DP, false>(c));
        const int vr = 4 * g + c / 4;
        const uint32_t v_at = lds_addr(stage) + vr * DP * 2 + (((c % 4) / 2 ^ v_swizzle<DP, false>(vr)) * 16) + (c & 1) * 8;
        const Tile& t = piece.t;
        const int head = piece.head, u0 = piece.u0, u1 = piece.u1, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const int begin = t.base + u0 * UNIT, end = min(t.hi, t.base + u1 * UNIT);
        const int blocks = end > begin ? (end - begin + kFewKeys - 1) / kFewKeys : 0;
        const int mine = (blocks - wave + WAVES - 1) / WAVES;  // blocks wave, wave + WAVES, ...
        auto first_of = [&](int i) { return begin + (wave + i * WAVES) * kFewKeys; };
        Key keys[2] = {};  // of the block that is loaded next, c and 16 + c
        auto find = [&](int i) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) keys[kt] = from.find(a, src, first_of(i) + kt * 16);
        };
        Quarter<DP> kq[2], vq[2];
        auto load = [&](const Key& key0, const Key& key1) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                from.load(a, src, src.k, kt ? key1 : key0, kq[kt]);
                from.load(a, src, src.v, kt ? key1 : key0, vq[kt]);
            }
        };
        if (mine > 0) find(0);
        u32x4 q[MT][KS];
        int row_lo[MT], row_hi[MT];  // keys that the lane's row sees
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            load_query<KS>(a, t, head, mt * 16 + c, g * KS, 1, q[mt]);
        }
        constexpr bool QLDS = kQueryInLds<DP, MT>;
        u32x4* const q_lds = reinterpret_cast<u32x4*>(smem + WAVES * kFewStage<DP>);
        if constexpr (QLDS) {  // operand (mt, st) of a lane: 64 lanes side by side
            static_assert(MT * KS % WAVES == 0, "the waves store as many each");
#pragma unroll
            for (int i = 0; i < MT * KS; ++i) {
                if (i % WAVES == wave) q_lds[i * 64 + lane] = q[i / KS][i % KS];
            }
            __syncthreads();
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int pos = t.first_pos + (t.row0 + mt * 16 + c) / a.group;
            row_hi[mt] = min(pos + 1, t.hi);
            row_lo[mt] = a.window > 0 ? pos + 1 - a.window : 0;
#pragma unroll
            for (int st = 0; st < KS && !QLDS; ++st) asm volatile("" : "+v"(q[mt][st]));  // here, not waited for in the loop
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
        if (mine > 0) {
            load(keys[0], keys[1]);
            if (mine > 1) find(1);
        }
        for (int i = 0; i < mine; ++i) {
            const int key0 = first_of(i);
            f32x4 s[MT][2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (QLDS) {
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    u32x4 qf[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) qf[mt] = q_lds[(mt * KS + st) * 64 + lane];
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        const u32x4 kf = widen<BF16, DP>(from.lane, kq[kt], st);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][kt] = mfma16x16x32<BF16>(kf, qf[mt], s[mt][kt]);
                    }
                }
            } else {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int st = 0; st < KS; ++st) {
                        const u32x4 kf = widen<BF16, DP>(from.lane, kq[kt], st);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][kt] = mfma16x16x32<BF16>(kf, q[mt][st], s[mt][kt]);
                    }
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                store_quarter<BF16, DP>(stage + kt * 16 * DP * 2, v_to, from.lane, vq[kt]);
            }
            if (i + 1 < mine) {  // the pages of the block after next ahead of the next one's codes: loads return in order
                const Key now0 = keys[0], now1 = keys[1];
                if (i + 2 < mine) find(i + 2);
                load(now0, now1);
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");  // a wave's LDS operations stay in this order
            const bool masked = key0 < all_lo || key0 + kFewKeys > all_hi;
            u32x4 p[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float x[8], top = -kInf;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[mt][e / 4][e % 4];
                cap_scores<CAP, 8, true>(a, x);
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = key0 + (e / 4) * 16 + 4 * g + e % 4;
                        x[e] = (key < row_lo[mt]) | (key >= row_hi[mt]) ? -kInf : x[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
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
            uint32_t v_now = v_at;
            asm volatile("" : "+v"(v_now));  // the tiles' places are computed, not held
            auto read_v = [&](int d) {
                u32x4 vf;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const u32x2 h = transposed<16 * DP * 2>(v_now ^ (d << 5), kt);
                    vf[2 * kt] = h[0];
                    vf[2 * kt + 1] = h[1];
                }
                return vf;
            };
            u32x4 vf[kAhead];
#pragma unroll
            for (int d = 0; d < kAhead; ++d) vf[d] = read_v(d);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) o[mt][d] = mfma16x16x32<BF16>(vf[d % kAhead], p[mt], o[mt][d]);
                if (d + kAhead < DT) vf[d % kAhead] = read_v(d + kAhead);
            }
            asm volatile("" ::: "memory");
        }
        __syncthreads();  // every wave is done with its stage
        join_waves<Fp4Keys, BF16, DP, MT, WAVES, CAP, MT>(a, t, smem, wave, head, slot, begin, end, k, m, z, o);
        __syncthreads();  // the stages are used again
    }
    clear_rest(a);
}

// ---- many rows --------------------------------------------------------------------

// Four waves of 32 query rows each over blocks of 64 keys that they share in LDS as 16-bit elements,
// two stages: each wave widens 16 keys of a block, whose codes came during the block before.  With two
// GROUPS of four waves, each with stages of its own, the blocks go to them in turn, and the second
// group's outputs reach the first one's through LDS at the end: for whole tiles too few to give a SIMD
// a second wave.
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;
template <int DP>
constexpr int kManyStage = 2 * kManyKeys * DP * 2;
template <int DP, int GROUPS>
constexpr int many_stage_bytes() {
    const int stages = GROUPS * 2 * kManyStage<DP>, join = kManyRows * (DP + 4) * 4;
    return GROUPS > 1 && join > stages ? join : stages;
}

template <bool BF16, int DP, bool CAP, int GROUPS>
__global__ __launch_bounds__(GROUPS * kManyWaves * 64) __attribute__((amdgpu_waves_per_eu(DP == 256 ? 1 : 2)))
void fp4_many_rows_kernel(const Fp4Params a) {
    constexpr int WAVES = kManyWaves, MR = kManyRows, KEYS = kManyKeys;
    constexpr int KS = DP / 16;      // steps of 16 head elements
    constexpr int DT = DP / 32;      // tiles of 32 output elements
    constexpr int COPY = KEYS / WAVES;
    static_assert(COPY == 16, "a load takes 16 keys");
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WAVES;
    const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WAVES : 0;
    const int c = lane & 31, h = lane >> 5;
    Plan& plan = *reinterpret_cast<Plan*>(smem + many_stage_bytes<DP, GROUPS>());
    uint8_t* const stages = smem + group * 2 * kManyStage<DP>;
    const Loader<DP> from(a, lane);
    const int copied = wave * COPY + (lane & 15);  // the lane's key of a block
    const uint32_t k_to = quarter_at<DP>(lane >> 4, copied, k_swizzle<DP>(copied));
    const uint32_t v_to = quarter_at<DP>(lane >> 4, copied, v_swizzle<DP, true>(copied));
    const float k = unit<CAP>(a);
    // LDS places of the lane's operands in a stage: K's unit 2 st + h of row c lies st << 5 (in
    // bits 5 up) away by XOR; V's 4 rows from 4 h on, at columns of tile d, d << 6 away
    const uint32_t k_at = (uint32_t)(c * DP * 2 + ((h ^ k_swizzle<DP>(c)) * 16));
    const int vr = 4 * h + ((c & 15) >> 2);
    const uint32_t v_at = (uint32_t)(kManyStage<DP> / 2 + vr * DP * 2 +
                                     ((((c >> 4) * 2 + ((c & 3) >> 1)) ^ v_swizzle<DP, true>(vr)) * 16) + (c & 1) * 8);
    Pieces<MR, KEYS, KEYS, GROUPS * WAVES, false, false, true> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        const Tile& t = piece.t;
        const int head = piece.head, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const int begin = t.base + piece.u0 * KEYS, end = min(t.hi, t.base + piece.u1 * KEYS);
        const int all = end > begin ? (end - begin + KEYS - 1) / KEYS : 0;
        const int rounds = (all + GROUPS - 1) / GROUPS, blocks = (all - group + GROUPS - 1) / GROUPS;  // the group's
        auto first_of = [&](int i) { return begin + (i * GROUPS + group) * KEYS; };
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
        Key key{};  // the lane's, of the block that is loaded next
        Quarter<DP> kq, vq;
        auto find = [&](int i) { return from.find(a, src, first_of(i) + wave * COPY); };
        auto load = [&] {
            from.load(a, src, src.k, key, kq);
            from.load(a, src, src.v, key, vq);
        };
        auto store = [&](int i) {
            uint8_t* const to = stages + (i & 1) * kManyStage<DP>;
            store_quarter<BF16, DP>(to, k_to, from.lane, kq);
            store_quarter<BF16, DP>(to + kManyStage<DP> / 2, v_to, from.lane, vq);
        };
        if (blocks > 0) {
            key = find(0);
            load();
            if (blocks > 1) key = find(1);
            store(0);
            if (blocks > 1) {
                load();
                if (blocks > 2) key = find(2);
            }
        }
        for (int i = 0; i < rounds; ++i) {
            // block i is there, and every wave is done with block i - 1
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (i + 1 < blocks) {
                store(i + 1);
                if (i + 2 < blocks) {
                    const Key then = i + 3 < blocks ? find(i + 3) : Key{};
                    load();
                    key = then;
                }
            }
            const int key0 = first_of(i);
            if (i >= blocks || !r.sees(key0)) continue;
            const uint8_t* const st_at = stages + (i & 1) * kManyStage<DP>;
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
            cap_scores<CAP, 16, true>(a, s[0]);
            cap_scores<CAP, 16, true>(a, s[1]);
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
                const uint8_t* const at_v = st_at + (v_at ^ ((n % DT) << 6)) + (n / DT) * 16 * DP * 2;
                const u32x2 y0 = read_transposed(at_v), y1 = read_transposed(at_v + 8 * DP * 2);
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
        }
        float held = held_max<BF16>(m, k);
        if constexpr (GROUPS > 1) {
            constexpr int kLane = 16 * DT + 2;  // floats of a lane: outputs, maximum, sum
            float* const theirs = reinterpret_cast<float*>(smem) + wave * kLane * 64 + lane;
            __syncthreads();  // every wave is done with the stages
            if (group == 1) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) theirs[(16 * d + e) * 64] = o[d][e];
                theirs[16 * DT * 64] = held;
                theirs[(16 * DT + 1) * 64] = z;
            }
            __syncthreads();
            if (group == 0) {
                const float m1 = theirs[16 * DT * 64], z1 = theirs[(16 * DT + 1) * 64], top = fmaxf(held, m1);
                // (a maximum of -inf: no key, or scores of NaN, which the sum has then)
                const float f0 = held == -kInf ? 0.f : __builtin_amdgcn_exp2f(held - top);
                const float f1 = m1 == -kInf ? 0.f : __builtin_amdgcn_exp2f(m1 - top);
                z = (held == -kInf ? z : f0 * z) + (m1 == -kInf ? z1 : f1 * z1);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        o[d][e] = (f0 == 0.f ? 0.f : f0 * o[d][e]) + (f1 == 0.f ? 0.f : f1 * theirs[(16 * d + e) * 64]);
                    }
                held = top;
            }
        }
        if (group == 0) {
            store_rows<Fp4Keys, BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held, z, o);
        }
        __syncthreads();  // every wave is done with the stages
    }
    clear_rest(a);
}

// ---- a great many rows -----------------------------------------------------------------

// Eight waves of 32 rows, two on each SIMD, that take turns: while waves 0 to 3 are in their products
// (scores of block i + 1, outputs of block i), waves 4 to 7 make the probabilities of a block, and the
// other way round (measured against waves without turns in paged_attention.hip).  Waves 0 to 3 widen K,
// waves 4 to 7 V, 16 keys each of a block, beside their probabilities; the codes come a block ahead.
constexpr int kWideWaves = 8, kWideRows = 32 * kWideWaves, kWideRing = 3;
template <int DP>
constexpr int kWideBlock = kManyKeys * DP * 2;  // bytes of K, or of V
template <int DP>
constexpr int wide_stage_bytes() { return 2 * kWideRing * kWideBlock<DP>; }

template <bool BF16, int DP, bool CAP>
__global__ __launch_bounds__(kWideWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void fp4_wide_rows_kernel(const Fp4Params a) {
    constexpr int MR = kWideRows, KEYS = kManyKeys, KS = DP / 16, DT = DP / 32;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // (nothing else is: it starts at 0)
    Plan& plan = *reinterpret_cast<Plan*>(smem + wide_stage_bytes<DP>());
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    const bool late = wave >= 4;  // half a turn behind, and widens V
    const Loader<DP> from(a, lane);
    const int copied = (wave & 3) * 16 + (lane & 15);  // the lane's key of a block
    uint8_t* const my_ring = smem + (late ? kWideRing * kWideBlock<DP> : 0);
    const uint32_t to = quarter_at<DP>(lane >> 4, copied, late ? v_swizzle<DP, true>(copied) : k_swizzle<DP>(copied));
    const float k = unit<CAP>(a);
    const uint32_t k_at = (uint32_t)(c * DP * 2 + ((h ^ k_swizzle<DP>(c)) * 16));
    const int vr = 4 * h + ((c & 15) >> 2);
    const uint32_t v_at = (uint32_t)(vr * DP * 2 + ((((c >> 4) * 2 + ((c & 3) >> 1)) ^ v_swizzle<DP, true>(vr)) * 16) +
                                     (c & 1) * 8);
    Pieces<MR, KEYS, KEYS, kWideWaves, false, false, true> piece;
    piece.start(a, plan);
    while (piece.next(a, plan)) {
        const Tile& t = piece.t;
        const int head = piece.head, slot = piece.slot;
        const Source src = source_of(a, t, head);
        const uint8_t* const plane = late ? src.v : src.k;
        const int begin = t.base + piece.u0 * KEYS, end = min(t.hi, t.base + piece.u1 * KEYS);
        const int blocks = end > begin ? (end - begin + KEYS - 1) / KEYS : 0;
        const WaveRows<KEYS> r(a, t, wave);
        const int mine0 = begin + (wave & 3) * 16;  // of block 0, the first key that the wave widens
        Quarter<DP> raw;
        Key key{};  // the lane's, of the block that is loaded next
        auto find = [&](int i) { return from.find(a, src, mine0 + i * KEYS); };
        auto load = [&] { from.load(a, src, plane, key, raw); };
        auto store = [&](int place) { store_quarter<BF16, DP>(my_ring + place * kWideBlock<DP>, to, from.lane, raw); };
        if (blocks > 0) key = find(0);
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
            // blocks 0 and 1 into the ring, block 2's codes and block 3's pages under way
            load();
            if (blocks > 1) key = find(1);
            store(0);
            if (blocks > 1) {
                load();
                if (blocks > 2) key = find(2);
                store(1);
            }
            if (blocks > 2) {
                load();
                if (blocks > 3) key = find(3);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (late) asm volatile("s_barrier" ::: "memory");
            int place = 2;  // ring place of block i + 3
            for (int i = -1; i < blocks; ++i) {
                // ---- products: scores of block i + 1, outputs of block i
                const int next = begin + (i + 1) * KEYS;
                const int place_next = place == 2 ? 0 : place + 1;  // of blocks i + 1 (and i + 4)
                const int place_now = place;                        // of blocks i (and i + 3)
                const bool do_next = i + 1 < blocks && r.sees(next), do_now = i >= 0 && r.sees(next - KEYS);
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
                // ---- block i + 3 into the ring, the codes of block i + 4; probabilities of block i + 1
                if (__builtin_expect(i + 3 < blocks, 1)) {
                    store(place_now);
                    if (i + 4 < blocks) {
                        const Key then = i + 5 < blocks ? find(i + 5) : Key{};
                        load();
                        key = then;
                    }
                }
                if (__builtin_expect(do_next, 1)) {
                    cap_scores<CAP, 16, true>(a, s[0]);
                    cap_scores<CAP, 16, true>(a, s[1]);
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
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                place = place_next;
            }
            if (!late) asm volatile("s_barrier" ::: "memory");
        }
        store_rows<Fp4Keys, BF16, DP, MR, CAP>(a, t, r, wave, head, slot, begin, end, held_max<BF16>(m, k), z, o);
        __syncthreads();  // every wave is done with the ring
    }
    clear_rest(a);
}

// ---- host ----------------------------------------------------------------------------

struct Call {
    Fp4Params p;
    int dp, tile_rows, grid;   // tile_rows: 16 or 32 (few rows), 128 or 256
    int groups;                // of 128 rows: of waves that share a tile's keys
    bool narrow;               // tiles of 32 rows where a sequence has several
    int plan;                  // bytes of LDS behind the kernel's stages
    int64_t pieces;            // split: that a tile's keys are in, about, the longest tile's
    int64_t tiles;             // at most
    size_t bytes;
};

int64_t page_bytes(const pw4_paged_attention_args* a) {
    return a->page_size * a->kv_heads * (a->head_dim / 2 + a->head_dim / 32);
}

// Which kernel, tiles and split, from what the host knows.  `a` has passed check().
Call plan_call(const pw4_paged_attention_args* a) {
    Call c{};
    Fp4Params& p = c.p;
    static_cast<Params&>(p) = params_of(a);
    p.page_bytes = (uint32_t)a->page_stride;
    p.row_codes = (uint32_t)(a->head_dim / 2);
    p.row_exps = (uint32_t)(a->head_dim / 32);
    p.head_codes = (uint32_t)a->page_size * p.row_codes;
    p.head_exps = (uint32_t)a->page_size * p.row_exps;
    p.exps_at = (uint32_t)a->kv_heads * p.head_codes;
    // (a power of two 2^n has 2^(31 - n) and 0; else as Params' division, with 2 key)
    p.index_magic = p.page_shift >= 0 ? 0x80000000u >> p.page_shift : p.page_magic;
    p.index_shift = p.page_shift >= 0 ? 0 : p.page_magic_shift + 1;
    const int64_t rows = (int64_t)p.max_q * p.group;
    c.dp = padded_dim(a->head_dim);
    const int cus = device_cus();
    const auto tiles_of = [&](int tile_rows) {
        return std::min(a->num_tokens * p.group / tile_rows + p.batch, p.batch * ceil_div(rows, tile_rows));
    };
    // keys that a tile's rows see at most: those that a window leaves, or all
    const auto keys_of = [&](int64_t tile_rows) {
        return p.window == 0 ? p.max_len
                             : std::min<int64_t>(p.max_len, (int64_t)p.window + (std::min(tile_rows, rows) + p.group - 2) / p.group);
    };
    // 256-row tiles run at the higher rate, but only one to a CU: for heads of 96 and 128 where they are long
    // and either fill the chip almost twice or, of chunks far into their sequences, are alike.  128 and 256
    // rows, us, 32 heads on 8 of 128: a prompt of 2048 tokens 62 and 71, of 4096 165 and 151, of 8192 584 and
    // 550, 16 of 512 83 and 97, 4 of 4000 in a window of 1024 305 and 318; 8 chunks of 1024 at 8000 keys, 8
    // heads, 300 and 259, a prompt of 8192 there 205 and 240.  (Heads of 64: 367 and 437 for a prompt of 8192;
    // three waves of 128-row tiles share a SIMD.)
    const int64_t wide_tiles = tiles_of(kWideRows) * p.kv_heads;
    const bool alike = p.max_len / 4 >= p.max_q;
    // 32-row tiles, whose waves have keys of their own, take less than half of 128-row tiles' time for one, but are
    // four times as many, each with the keys to widen: for up to two a CU, over keys that are enough to tell and
    // too few to split 128-row tiles for.  32 and 128 rows (those whole or split, as below), us, heads of 64 / 128:
    //   18 tiles (6) of 300 keys 13.3 and 12.1 / 16.8 and 15.8, of 450 14.2 and 14.8 / 17.8 and 19.7, of 1200 18.9 and
    //   23.9 / 24 and 31, of 2400 25.6 and 24.4 / 33 and 31; 252 (84) of 1200 19.6 and 25.5 / 25 and 35, of 3200 32 and
    //   39 / 42 and 50, of 4000 38 and 42 / 50 and 54; 324 (108) of 800 21.0 and 20.8 / 27 and 28, of 2400 35 and 44 /
    //   47 and 66, of 4000 51 and 49 / 65 and 64; 512 (128) of 1200 24.7 and 25.8 / 32 and 35, of 4000 50 and 54 / 65
    //   and 71, of 6000 68 and 66 / 87 and 88; 576 (144) of 2400 44 and 43 / 70 and 64
    const int64_t narrow_tiles = tiles_of(32) * p.kv_heads, narrow_keys = keys_of(32);
    bool narrow = narrow_tiles <= cus ? narrow_keys >= 400 && (narrow_keys - 2048) * cus <= 2304 * narrow_tiles
                                      : narrow_tiles <= 2 * cus && narrow_keys >= 1000 &&
                                            (narrow_keys - 1280) * cus <= 1664 * narrow_tiles;
    const char* const forced_tile = plan_override("PW4_ATTN_TILE");
    if (forced_tile) narrow = forced_tile[0] == '3';
    narrow = narrow && rows > 32 && c.dp != 256;
    c.tile_rows = rows <= 16 ? 16 : rows <= 32 || narrow ? 32
                  : c.dp == 128 && 4 * wide_tiles >= (alike ? 4 : 7) * cus && keys_of(kWideRows) >= 24 * kManyKeys ? kWideRows
                                                                                                                  : kManyRows;
    if (forced_tile && c.tile_rows > 32 && c.dp == 128) c.tile_rows = forced_tile[0] == '2' ? kWideRows : kManyRows;
    const bool few = c.tile_rows <= 32;
    c.narrow = narrow;
    c.tiles = few && !narrow ? p.batch : tiles_of(c.tile_rows);
    const int unit = !few ? kManyKeys : c.dp == 64 ? kFewUnit<64> : c.dp == 128 ? kFewUnit<128> : kFewUnit<256>;
    // what a split call holds in LDS: a plan, or the tiles of few sequences
    c.plan = !few || p.batch > 64 ? (int)sizeof(Plan) : 64 * (int)sizeof(Tile);
    // workgroups that run at once
    const auto few_at_once = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        return c.dp == 64 ? few_slots<64, MT>(c.plan) : c.dp == 128 ? few_slots<128, MT>(c.plan) : few_slots<256, MT>(c.plan);
    };
    const int slots = cus * (c.tile_rows == 16   ? few_at_once(std::integral_constant<int, 1>{})
                             : c.tile_rows == 32 ? few_at_once(std::integral_constant<int, 2>{})
                             : c.tile_rows == kManyRows && c.dp != 256 ? 2
                                                                       : 1);
    const int64_t most_units = ceil_div(keys_of(c.tile_rows), unit) + 1;  // of a tile
    const char* const forced = plan_override("PW4_ATTN_UNITS");
    const int forced_units = forced ? std::atoi(forced) : 0;
    // A few rows: pieces of one unit make long joins of long sequences.  Pieces of 1 and 4 units (16 waves to join,
    // below), us, 4 query heads on each of 2 key-value heads of 128: 65000 keys 27 and 18.4, six tokens there 37 and
    // 26; one head, 131072 keys 36 and 20; 8 heads, 16000 keys 21.7 and 17.6; of 3 units, 8000 keys 15.4 and 14.1,
    // 6000 15.1 and 16.4.
    p.min_units = forced_units > 0 ? forced_units : !few ? 8 : most_units > 96 ? 4 : most_units > 50 ? 3 : 1;
    // Whether the keys are split.  A few rows: whole, a workgroup takes 0.5, 0.7 and 1.3 us a unit (heads of
    // 64 and 128, units of 128 keys; of 256, of 64); the split, a second launch, and the partial outputs' way
    // through memory, which grow with the tiles.  8 key-value heads, sequences of one length, whole and split, us:
    // (the rule splits the first, of 1100 keys, for 0.7 us more)
    //   heads of 64   1 of 1100 keys 9.5 and 10.2, of 1600 11.6 and 10.2; 8 of 2400 15.3 and 15.3, of 4000 22 and 17;
    //                 32 of 4000 27 and 29
    //   heads of 128  1 of 777 10.4 and 11.0, of 1100 12.0 and 11.1; 8 of 1600 15.6 and 15.5, of 4000 32 and 19;
    //                 16 of 2400 22 and 24, of 4000 33 and 24; 32 of 6000 48 and 48, of 8000 68 and 59
    //   heads of 256  1 of 200 11.8 and 13.2, of 400 15.5 and 13.1; 16 of 777 23 and 25, of 1100 30 and 24
    // Many rows: the longest tile against the work's share of a place, the join and the partial outputs.  Heads of
    // 128, tiles of all heads and their keys, whole and split, us: 6 of 777 26 and 31, of 8000 172 and 34; 48 of 4000
    // 96 and 50; 88 of 1000 31 and 43; 128 of 4000 98 and 70; 176 of 5000 119 and 100; 224 of 1000 31 and 61.
    const int64_t work = c.tiles * p.kv_heads;
    const char* const forced_split = plan_override("PW4_ATTN_SPLIT");
    const bool wanted = forced_split ? forced_split[0] == '1'
                        : few ? most_units > (c.dp == 256 ? 5 + 20 * work / cus : 9 + 28 * work / cus)
                              : most_units * (slots - work) > slots * (c.dp == 256 ? 14 + work / 16 : 16 + work / 7);
    // Whole tiles of 128 rows that leave CUs idle: two groups of waves.  One and two, us, heads of 64 / 128: 6 tiles of
    // 300 keys 12.0 and 13.4 / 15.8 and 18.0, of 777 20.0 and 19.5 / 26.8 and 26.6; 132 of 1500 30.7 and 26.8 / 42 and
    // 38; 176 of 2000 39 and 33 / 55 and 48, of 5000 81 and 65 / 116 and 95; more than CUs, 336 of 1500, 42 and 50 / 61
    // and 73.
    const char* const forced_groups = plan_override("PW4_ATTN_GROUPS");
    c.groups = c.tile_rows != kManyRows || c.dp == 256 ? 1
               : forced_groups                         ? forced_groups[0] - '0'
               : !wanted && work <= cus && keys_of(kManyRows) >= 900 ? 2
                                                                      : 1;
    p.split = wanted && c.groups == 1 && !narrow && c.tiles > 0 && p.batch <= kMaxSplitTiles && c.tiles <= kMaxSplitTiles &&
              c.tiles * p.kv_heads * most_units < INT_MAX;
    if (!p.split) c.plan = 0;
    c.grid = (int)(c.tiles * p.kv_heads);
    // (6 chunks in a window of 1024, 270 tiles, those of the fifth chunk a third as long: 38 us, in the sequences'
    // order 50)
    p.order = p.batch > 1 && p.batch <= 64 && c.grid > cus;
    if (p.split) {
        c.grid = (int)std::min<int64_t>(slots, ceil_div(c.tiles * p.kv_heads * most_units, p.min_units));
        c.bytes = partial_bytes(c.grid, c.tile_rows, p.dim);
        c.pieces = most_units / std::max<int64_t>(p.min_units, c.tiles * p.kv_heads * most_units / c.grid);
    }
    return c;
}

template <bool BF16, int DP, bool CAP>
hipError_t launch(const Call& c, hipStream_t s) {
    hipError_t e;
    if (c.tile_rows == 16) {
        e = run_attention<fp4_few_rows_kernel<BF16, DP, 1, CAP, true>>(c.p, c.grid, kFewWaves<DP>, few_stage_bytes<DP, 1>(), c.plan, s);
    } else if (c.tile_rows == 32 && !c.narrow) {
        e = run_attention<fp4_few_rows_kernel<BF16, DP, 2, CAP, true>>(c.p, c.grid, kFewWaves<DP>, few_stage_bytes<DP, 2>(), c.plan, s);
    } else if (c.tile_rows == 32) {
        if constexpr (DP != 256) {
            e = run_attention<fp4_few_rows_kernel<BF16, DP, 2, CAP, false>>(c.p, c.grid, kFewWaves<DP>, few_stage_bytes<DP, 2>(), 0, s);
        } else {
            e = hipErrorInvalidValue;  // no such tile: plan_call
        }
    } else if (c.tile_rows == kManyRows) {
        if (c.groups == 1 || DP == 256) {
            e = run_attention<fp4_many_rows_kernel<BF16, DP, CAP, 1>>(c.p, c.grid, kManyWaves, many_stage_bytes<DP, 1>(), c.plan, s);
        } else {
            constexpr int G = DP < 256 ? 2 : 1;
            e = run_attention<fp4_many_rows_kernel<BF16, DP, CAP, G>>(c.p, c.grid, G * kManyWaves, many_stage_bytes<DP, G>(), c.plan, s);
        }
    } else if constexpr (DP == 128) {
        e = run_attention<fp4_wide_rows_kernel<BF16, DP, CAP>>(c.p, c.grid, kWideWaves, wide_stage_bytes<DP>(), c.plan, s);
    } else {
        e = hipErrorInvalidValue;  // no such tile: plan_call
    }
    if (e != hipSuccess || !c.p.split) return e;
    const int rows = (int)std::max<int64_t>(1, std::min<int64_t>(c.tile_rows, (int64_t)c.p.max_q * c.p.group));
    // A wave a row to join where rows are enough, a workgroup where not.  Both launches, workgroup and wave, us,
    // heads of 128: 16 tokens over 2 to 32 thousand keys (512 rows) 46 and 48, two of each 48 and 50, four (2048) 54
    // and 53, eight 76 and 72, eight of 48 sequences 173 and 156, one of each (1536) 128 and 125; eight of 2 sequences
    // (512) 45 and 55.  Sixteen waves to that workgroup where a tile is in many pieces: 131072 keys of one head in
    // 256 20 and with four waves 28, 65000 of two in 127 18.4 and 20.9; 16000 of eight in 31 18.7 and 17.6.
    const bool long_joins = c.pieces > 48;
    const bool wave_a_row = rows * c.tiles * c.p.kv_heads >= 6 * device_cus();
    if (c.tile_rows == 16) {
        wave_a_row   ? run_join<16, BF16>(c.p, c.tiles, c.grid, s)
        : long_joins ? run_row_join<16, BF16, 16>(c.p, c.tiles, rows, c.grid, s)
                     : run_row_join<16, BF16, 4>(c.p, c.tiles, rows, c.grid, s);
    } else if (c.tile_rows == 32) {
        wave_a_row   ? run_join<32, BF16>(c.p, c.tiles, c.grid, s)
        : long_joins ? run_row_join<32, BF16, 16>(c.p, c.tiles, rows, c.grid, s)
                     : run_row_join<32, BF16, 4>(c.p, c.tiles, rows, c.grid, s);
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
    if (a->head_dim % 32 != 0) return PW4_ERR_SHAPE;
    if (a->num_tokens == 0) return PW4_OK;
    const uint64_t addresses = (uint64_t)(uintptr_t)a->q | (uint64_t)(uintptr_t)a->k_cache |
                               (uint64_t)(uintptr_t)a->v_cache | (uint64_t)(uintptr_t)a->out;
    if ((addresses & 15) != 0 || ((a->q_token_stride | a->q_head_stride) & 7) != 0) return PW4_ERR_ARG;
    if (a->kv_heads > 65535 || a->page_size > INT_MAX / 256 / a->kv_heads) return PW4_ERR_SHAPE;
    if (a->page_stride < 0 || a->page_stride % 16 != 0) return PW4_ERR_ARG;
    if (a->page_stride > INT_MAX || (a->num_pages > 1 && a->page_stride < page_bytes(a))) return PW4_ERR_SHAPE;
    return PW4_OK;
}

}  // namespace

extern "C" {

size_t pw4_paged_attention_fp4_workspace_size(const pw4_paged_attention_args* args) {
    return check(args) != PW4_OK || args->num_tokens == 0 ? 0 : plan_call(args).bytes;
}

int pw4_paged_attention_fp4(const pw4_paged_attention_args* args, void* workspace, size_t workspace_bytes,
                            pw4_stream_t stream) {
    if (const int rc = check(args)) return rc;
    if (args->num_tokens == 0) return PW4_OK;
    Call c = plan_call(args);
    const int waves = c.tile_rows > kManyRows ? kWideWaves : c.tile_rows > 32 ? c.groups * kManyWaves
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

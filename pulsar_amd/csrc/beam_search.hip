// Beam search's selection and the reordering of the beams' states (the definitions:
// pulsar_paged.h).
//
// Bound by one read of the logits: a row's slices are read once, as token_logprobs reads them,
// and leave their largest logit, sum e^(x-m) and `width` best candidates.  The second launch has
// a workgroup a search, whose waves join a beam's slices each: its log-sum-exp, the slices'
// sums added in fp64, and its best candidates in order.  No beam gives more than `width` of the
// new ones, so width times beams candidates are left, in lists that fall by total, which are
// merged pair by pair: a candidate's place in the merged list is its own and, by bisection,
// how many of the other list are ahead.  Totals are fp64: scores of some hundred tokens have fp32
// steps of 1e-5, within which beams would tie.  A slice's e^(x-m) and their sum are fp32, as the
// hardware's exponential is (the first launch is the one that its instructions weigh on): that is some units
// of 2^-24 of a row's sum, the same for all of its candidates, and for equal rows.
//
// 32 searches of 8 beams, a fifth of them ended, over 100003 bf16 logits (41 MB) take 14 us for the first
// launch (3.0 TB/s; vector units busy 36% of the cycles, waves waiting 52%), 7.3 for the second and 3.7 to
// reorder 500 tokens a beam; 24 a call of both.  The second launch is a chain of steps by one workgroup a search, waves
// waiting 83% of their time; one that ranked every candidate against all others took 111 us for 32
// beams, merging 34, and with the lists made in a launch of their own 26, all three launches and the
// reordering.
#include "logit_slices.h"

#include <type_traits>

using namespace pw4;

namespace {

constexpr int kMaxBeams = 32;
constexpr int kWaves = 16;  // of the second launch, a wave a beam

struct SelectArgs {
    SliceArgs s;
    const float* scores;
    int64_t end_token;
    float* out_scores;
    int32_t* out_rows;
    int64_t* out_tokens;
    uint8_t* out_ended;
    double* totals;    // workspace [rows, width], more than kWaves beams: the beams' lists
    uint64_t* keys;
    int32_t beams, width;
};

constexpr double kLowest = -__builtin_inf();

// ln sum e^x of a row, by a wave; NaN where the row has a NaN or +inf, -inf where it is all -inf.
__device__ __forceinline__ double join_lse(const SliceSums* sums, int slices) {
    const int lane = threadIdx.x & 63;
    float m = -__builtin_inff();
    for (int s = lane; s < slices; s += 64) m = fmaxf(m, sums[s].m);
    m = wave_max(m);
    double z = 0;
    for (int s = lane; s < slices; s += 64) {
        const SliceSums p = sums[s];
        if (p.m == -__builtin_inff() && p.z == p.z) continue;
        z += p.z * exp((double)p.m - (double)m);
    }
    z = wave_sum(z);
    return (double)m + log(z);
}

// A list of candidates, best first: totals, and which candidate each is.
struct Lists {
    double total[kMaxBeams * kMaxTop];
    int which[kMaxBeams * kMaxTop];
    int length[kMaxBeams];
};

// Beam `row`'s continuations as a list, by a wave: totals and keys of logit and token, best first.  Returns
// the list's length.
template <int JOIN>
__device__ __forceinline__ int make_list(const SelectArgs& a, int row, uint64_t* join, double* totals, uint64_t* keys) {
    const int lane = threadIdx.x & 63, per = a.s.top_k;
    const double score = a.scores[row];
    const SliceSums* const sums = a.s.sums + (int64_t)row * a.s.slices;
    const uint64_t* const tops = a.s.top + (int64_t)row * a.s.slices * per;
    // one trip to memory: the lines that the steps below read one after the other
    const uint64_t line = tops[min(lane * 16, a.s.slices * per - 1)];
    const float sum = sums[min(lane, a.s.slices - 1)].m;
    const bool passed = a.s.passed != nullptr && a.s.passed[row] != 0;
    asm volatile("" ::"v"(line), "v"(sum));
    if (passed) {
        if (lane == 0) totals[0] = score == score ? score : kLowest;
        return 1;
    }
    const double lse = join_lse(sums, a.s.slices);
    join_tops<JOIN>(tops, a.s.slices, per, join, [&](int place, uint64_t key) {
        const double total = score + ((double)unordered((uint32_t)(key >> 32)) - lse);
        keys[place] = key;
        totals[place] = total == total ? total : kLowest;
    });
    return per;
}

// The lists of more beams than a workgroup has waves, a wave a list, to the workspace: with two lists a
// wave, each a chain of loads behind the last, 32 beams of 32003 logits took 21 us in one workgroup; with
// this launch 7 and 7.
__global__ __launch_bounds__(kThreads) void list_kernel(const SelectArgs a) {
    __shared__ uint64_t s_join[kThreads / 64][kJoin];
    const int row = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (row >= a.s.tokens) return;
    make_list<kJoin>(a, row, s_join[threadIdx.x >> 6], a.totals + (int64_t)row * a.width, a.keys + (int64_t)row * a.width);
}

// A search's lists, made here (a wave a beam) or read, MADE, from the workspace, become one.
template <int WAVES, bool MADE>
__global__ __launch_bounds__(WAVES * 64) void select_kernel(const SelectArgs a) {
    constexpr int JOIN = MADE ? 1 : WAVES > 4 ? 128 : kJoin;
    __shared__ uint64_t s_join[WAVES][JOIN];
    __shared__ uint64_t s_key[kMaxBeams * kMaxTop];
    __shared__ Lists s_lists[2];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int row0 = blockIdx.x * a.beams;
    if constexpr (MADE) {
        Lists& l = s_lists[0];
        for (int i = tid; i < a.beams * a.width; i += WAVES * 64) {
            const int64_t at = (int64_t)row0 * a.width + i;
            l.total[i] = a.totals[at];
            l.which[i] = i;
            s_key[i] = a.keys[at];
        }
        if (tid < a.beams) l.length[tid] = a.s.passed != nullptr && a.s.passed[row0 + tid] != 0 ? 1 : a.s.top_k;
    } else {
        Lists& l = s_lists[0];
        for (int k = wave; k < a.beams; k += WAVES) {
            const int at = k * a.width, length = make_list<JOIN>(a, row0 + k, s_join[wave], l.total + at, s_key + at);
            for (int i = tid & 63; i < a.width; i += 64) l.which[at + i] = at + i;
            if ((tid & 63) == 0) l.length[k] = length;
        }
    }
    // Neighbouring lists become one, of `width` candidates at most, until one is left: a candidate's
    // place there is its own and how many of the other list are ahead of it.
    int from = 0;
    for (int lists = a.beams; lists > 1; lists = (lists + 1) / 2, from ^= 1) {
        const Lists& l = s_lists[from];
        Lists& to = s_lists[from ^ 1];
        __syncthreads();
        for (int i = tid; i < lists * a.width; i += WAVES * 64) {
            const int list = i / a.width, place = i - list * a.width, other = list ^ 1;
            if (place >= l.length[list]) continue;
            const double total = l.total[i];
            int lo = 0, hi = other < lists ? l.length[other] : 0;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double t = l.total[other * a.width + mid];
                if (t > total || (t == total && other < list)) {
                    lo = mid + 1;
                } else {
                    hi = mid;
                }
            }
            if (place + lo < a.width) {
                const int dst = (list >> 1) * a.width + place + lo;
                to.total[dst] = total;
                to.which[dst] = l.which[i];
            }
        }
        for (int i = tid; i < (lists + 1) / 2; i += WAVES * 64) {
            to.length[i] = min(a.width, l.length[2 * i] + (2 * i + 1 < lists ? l.length[2 * i + 1] : 0));
        }
    }
    __syncthreads();
    if (tid < min(a.width, s_lists[from].length[0])) {
        const int which = s_lists[from].which[tid], row = row0 + which / a.width;
        const bool ended = a.s.passed != nullptr && a.s.passed[row] != 0;
        const int64_t at = (int64_t)blockIdx.x * a.width + tid;
        const int64_t token = ended ? a.end_token : (int64_t)(uint32_t)~s_key[which];
        a.out_scores[at] = (float)s_lists[from].total[tid];
        a.out_rows[at] = row;
        a.out_tokens[at] = token;
        if (a.out_ended != nullptr) a.out_ended[at] = ended || token == a.end_token;
    }
}

// ---- reordering -----------------------------------------------------------------

constexpr int kStates = 8;            // of a launch
// Bytes of a row that a workgroup copies.  4096, 16384 and 65536, us: 256 histories of 500 tokens 2.4, 2.4 and 2.4, of
// 4096 4.1, 3.9 and 4.4; 4 states of 1 MB 3.0, 3.2 and 5.0; 32 of 512 KB 6.7, 5.8 and 8.3, of 8 MB 90, 95 and 104.
constexpr int64_t kPiece = 16384;

struct ReorderArgs {
    const uint8_t* src[kStates];
    uint8_t* dst[kStates];
    int64_t row_bytes[kStates], num_rows[kStates];
    int32_t pieces[kStates];          // of a row
    int64_t end[kStates];             // ascending sums of n * pieces
    const int32_t* rows;
    int32_t count;
    uint8_t width[kStates];           // bytes that a thread copies at once: 16, 8, 4, 2 or 1
};

template <typename V>
__device__ __forceinline__ void copy_as(const uint8_t* from, uint8_t* to, int64_t bytes, bool there) {
    const V* const f = reinterpret_cast<const V*>(from);
    V* const t = reinterpret_cast<V*>(to);
    for (int e = threadIdx.x; e < bytes / (int)sizeof(V); e += kThreads) t[e] = there ? f[e] : V{};
}
// A row's piece of a state: 16 KB a workgroup, so that short rows of many beams and long rows of few
// both spread.  Each state goes by the width that its own rows and addresses allow: 256 MB
// of states, alone, beside a flag of a byte a row, and beside histories of 501 tokens, take 95 us, 95 and 95; by
// the least width of all states of a launch 95, 294 and 120.  VECTORS: 16 bytes for all of them (256 histories of
// 500 tokens 2.40 us, where the kernel that looks the width up takes 2.52; 16 MB of states 5.74 and 5.86).
template <bool VECTORS>
__device__ __forceinline__ void copy_piece(const ReorderArgs& a, int64_t piece) {
    int s = 0;
    while (s + 1 < a.count && piece >= a.end[s]) ++s;
    const int64_t item = piece - (s ? a.end[s - 1] : 0);
    const int64_t i = item / a.pieces[s], begin = (item - i * a.pieces[s]) * kPiece;
    const int64_t row = a.rows[i];
    const int64_t bytes = min(kPiece, a.row_bytes[s] - begin);
    const int width = VECTORS ? 16 : a.width[s];
    const bool there = row >= 0 && row < a.num_rows[s];
    const uint8_t* const from = a.src[s] + (there ? row : 0) * a.row_bytes[s] + begin;
    uint8_t* const to = a.dst[s] + i * a.row_bytes[s] + begin;
    if (width == 16) {
        copy_as<u32x4>(from, to, bytes, there);
    } else if (width == 8) {
        copy_as<u32x2>(from, to, bytes, there);
    } else if (width == 4) {
        copy_as<uint32_t>(from, to, bytes, there);
    } else if (width == 2) {
        copy_as<uint16_t>(from, to, bytes, there);
    } else {
        copy_as<uint8_t>(from, to, bytes, there);
    }
}
template <bool VECTORS>
__global__ __launch_bounds__(kThreads) void reorder_kernel(const ReorderArgs a) {
    for (int64_t piece = blockIdx.x; piece < a.end[a.count - 1]; piece += gridDim.x) copy_piece<VECTORS>(a, piece);
}

}  // namespace

extern "C" {

size_t pw4_beam_select_workspace_size(int64_t batch, int64_t beams, int64_t vocab, int64_t width) {
    if (batch <= 0 || beams <= 0 || beams > kMaxBeams || batch > 65535 / beams || vocab <= 0 || vocab > INT_MAX / 2 ||
        width <= 0 || width > kMaxTop) {
        return 0;
    }
    const int64_t rows = batch * beams, slices = slices_of(rows, vocab);
    return sums_bytes(rows, slices) + (size_t)(rows * slices * std::min(width, vocab)) * 8 +
           (beams > kWaves ? (size_t)(rows * width) * 16 : 0);
}

int pw4_beam_select(const void* logits, int dtype, int64_t batch, int64_t beams, int64_t vocab, int64_t row_stride,
                    const float* scores, const uint8_t* ended, int64_t end_token, int64_t width, float* out_scores,
                    int32_t* out_rows, int64_t* out_tokens, uint8_t* out_ended, void* workspace,
                    size_t workspace_bytes, pw4_stream_t stream) {
    if (batch < 0 || beams <= 0 || vocab <= 0 || width <= 0) return PW4_ERR_ARG;
    if (dtype != PW4_DTYPE_F16 && dtype != PW4_DTYPE_BF16 && dtype != PW4_DTYPE_F32) return PW4_ERR_ARG;
    if (ended != nullptr && (end_token < -1 || end_token >= vocab)) return PW4_ERR_ARG;
    if (beams > kMaxBeams || width > kMaxTop || vocab > INT_MAX / 2 || batch > 65535 / beams || width > beams * vocab ||
        (ended != nullptr && width > beams) || row_stride < vocab) {
        return PW4_ERR_SHAPE;
    }
    if (batch == 0) return PW4_OK;
    if (!logits || !scores || !out_scores || !out_rows || !out_tokens || (out_ended != nullptr && ended == nullptr)) return PW4_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == PW4_DTYPE_F32 ? 4 : 2) != 0) return PW4_ERR_ARG;
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
        workspace_bytes < pw4_beam_select_workspace_size(batch, beams, vocab, width)) {
        return PW4_ERR_WORKSPACE;
    }
    const int64_t rows = batch * beams;
    const int slices = slices_of(rows, vocab);
    const SliceArgs slicing{logits, nullptr, ended, static_cast<SliceSums*>(workspace),
                            reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) + sums_bytes(rows, slices)),
                            row_stride, (int32_t)rows, (int32_t)vocab, (int32_t)std::min(width, vocab), slices,
                            (int32_t)ceil_div(vocab, slices)};
    double* const totals = reinterpret_cast<double*>(slicing.top + rows * slices * slicing.top_k);
    const SelectArgs a{slicing, scores, end_token, out_scores, out_rows, out_tokens, out_ended, totals,
                       reinterpret_cast<uint64_t*>(totals + rows * width), (int32_t)beams, (int32_t)width};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid(slices, (unsigned)rows);
    const auto run = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (per_thread(rows, vocab) == 16) {
            hipLaunchKernelGGL((slice_kernel<DT, 16, false>), grid, dim3(kThreads), 0, s, slicing);
        } else {
            hipLaunchKernelGGL((slice_kernel<DT, 32, false>), grid, dim3(kThreads), 0, s, slicing);
        }
    };
    if (dtype == PW4_DTYPE_F16) {
        run(std::integral_constant<int, PW4_DTYPE_F16>{});
    } else if (dtype == PW4_DTYPE_BF16) {
        run(std::integral_constant<int, PW4_DTYPE_BF16>{});
    } else {
        run(std::integral_constant<int, PW4_DTYPE_F32>{});
    }
    // Up to four beams: workgroups of four waves.  Four and sixteen, us of all launches: one beam of 128000 logits 7.2
    // and 7.5, four 9.2 and 9.2, four of 1000 8.8 and 9.3, 32 searches of one of 32003 7.9 and 8.0.
    if (beams <= 4) {
        hipLaunchKernelGGL((select_kernel<4, false>), dim3((unsigned)batch), dim3(4 * 64), 0, s, a);
    } else if (beams <= kWaves) {
        hipLaunchKernelGGL((select_kernel<kWaves, false>), dim3((unsigned)batch), dim3(kWaves * 64), 0, s, a);
    } else {
        hipLaunchKernelGGL(list_kernel, dim3((unsigned)ceil_div(rows, kThreads / 64)), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL((select_kernel<kWaves, true>), dim3((unsigned)batch), dim3(kWaves * 64), 0, s, a);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

int pw4_beam_reorder(const pw4_beam_state* states, int64_t count, const int32_t* rows, int64_t n,
                     pw4_stream_t stream) {
    if (count < 0 || n < 0 || (count && !states)) return PW4_ERR_ARG;
    if (n > INT_MAX) return PW4_ERR_SHAPE;
    for (int64_t i = 0; i < count; ++i) {
        const pw4_beam_state& st = states[i];
        if (st.row_bytes < 0 || st.num_rows < 0) return PW4_ERR_ARG;
        if (st.num_rows > INT_MAX || (st.row_bytes - 1) / kPiece + 1 > INT_MAX / kStates / std::max<int64_t>(n, 1)) return PW4_ERR_SHAPE;
        if (n && st.row_bytes && (!rows || !st.dst || (st.num_rows && !st.src))) return PW4_ERR_ARG;
    }
    if (n == 0) return PW4_OK;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    for (int64_t first = 0; first < count;) {
        ReorderArgs a{};
        a.rows = rows;
        int64_t items = 0;
        bool vectors = true;
        for (; first < count && a.count < kStates; ++first) {
            const pw4_beam_state& st = states[first];
            if (st.row_bytes == 0) continue;
            const int c = a.count++;
            a.src[c] = static_cast<const uint8_t*>(st.src);
            a.dst[c] = static_cast<uint8_t*>(st.dst);
            a.row_bytes[c] = st.row_bytes;
            a.num_rows[c] = st.num_rows;
            a.pieces[c] = (int32_t)ceil_div(st.row_bytes, kPiece);
            a.end[c] = items += n * a.pieces[c];
            const uint64_t all = (uint64_t)(uintptr_t)st.src | (uint64_t)(uintptr_t)st.dst | (uint64_t)st.row_bytes | 16;
            a.width[c] = (uint8_t)(all & -all);  // the lowest bit
            vectors &= a.width[c] == 16;
        }
        if (a.count == 0) break;
        const dim3 grid((unsigned)std::min<int64_t>(items, 1 << 22));  // (2^32 threads are too many)
        if (vectors) {
            hipLaunchKernelGGL(reorder_kernel<true>, grid, dim3(kThreads), 0, s, a);
        } else {
            hipLaunchKernelGGL(reorder_kernel<false>, grid, dim3(kThreads), 0, s, a);
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return report_hip_error(e);
    }
    return PW4_OK;
}

}  // extern "C"

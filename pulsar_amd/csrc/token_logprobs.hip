// Log probabilities of given tokens, with rank, entropy and top alternatives.
//
// Bound by one read of the logits.  A row is cut into slices, one workgroup of 256
// threads each, which holds its slice in registers, packed as it came: 32 logits a
// thread (2048 tokens of 100003 bf16 logits took 188 us so, and 64 a thread, at five waves
// a SIMD instead of eight, 206), or 16 where the tokens are so few that CUs would be idle.  The
// largest logit, then sum e^(x-m) and sum e^(x-m) (x-m) with the slice's own m, the rank
// and the top candidates come from one trip to memory.  A second launch joins a row's
// slices, a wave a row: with M = max m and the slices' sums scaled by e^(m-M),
//   lse = M + ln Z,  entropy = ln Z - T / Z,  Z = sum e^(x-M), T = sum e^(x-M) (x-M)
//
// Top candidates.  A number that the largest logits of at least k of 64 groups reach
// (four threads a group) is a bound that at least k logits reach, and few more: those
// are listed in LDS and ranked against each other.  Where ties make the list longer than
// it holds, those above the exact bound and the first k that equal it are; failing that,
// k rounds of a workgroup-wide maximum find the same tokens.
//
// 2048 tokens of 100003 bf16 logits (410 MB) take 160 us and 8.6 for the join under a
// profiler, 164 a call (2.5 TB/s): bound by the vector units, busy 74% of the first
// launch's cycles, which spend about 21 instructions on a logit (unpacking
// twice, the maximum, six for the sums with one transcendental, the rank's two where a
// vector holds a logit that is ahead).
//
// A row may begin at any address: vectors cover the 16-byte aligned part of a slice, and
// what is before and behind it, 14 logits at most, are the first threads' odd ones.
#include "logit_slices.h"

using namespace pw4;

namespace {

struct LogprobArgs {
    SliceArgs s;
    float* logprobs;
    int64_t* ranks;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
};

// One wave a row.
template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(const LogprobArgs a) {
    __shared__ uint64_t s_keys[kThreads / 64][kJoin];
    const int row = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.s.tokens) return;
    const SliceSums* const sums = a.s.sums + (int64_t)row * a.s.slices;
    constexpr float kInf = __builtin_inff(), kLog2e = 1.4426950408889634f;
    float m = -kInf;
    for (int s = lane; s < a.s.slices; s += 64) m = fmaxf(m, sums[s].m);
    m = wave_max(m);
    float z = 0.f, t = 0.f;
    int ahead = 0;
    for (int s = lane; s < a.s.slices; s += 64) {
        const SliceSums p = sums[s];
        ahead += p.ahead;
        if (p.m == -kInf && p.z == p.z) continue;
        const float d = fmaxf(p.m - m, -1e30f), w = __builtin_amdgcn_exp2f(d * kLog2e);  // 0 * -inf is no term
        z += p.z * w;
        t += (p.t + d * p.z) * w;
    }
    z = wave_sum(z);
    t = wave_sum(t);
    ahead = wave_sum(ahead);
    const bool empty = m == -kInf && z == 0.f;
    const float log_z = logf(z);
    auto logprob = [&](float x) { return empty ? -kInf : (x - m) - log_z; };
    if (lane == 0) {
        const int64_t target = a.s.targets[row];
        const bool given = target >= 0 && target < a.s.vocab;
        const int64_t at = (int64_t)row * a.s.row_stride * (DT == PW4_DTYPE_F32 ? 4 : 2);
        const float x = given ? logit_at<DT>(static_cast<const uint8_t*>(a.s.logits) + at, target) : 0.f;
        a.logprobs[row] = given ? logprob(x) : 0.f;
        a.ranks[row] = given ? ahead : -1;
        a.entropy[row] = empty ? 0.f : log_z - t / z;
    }
    if (a.s.top_k == 0) return;
    const uint64_t* const tops = a.s.top + (int64_t)row * a.s.slices * a.s.top_k;
    auto store = [&](int place, uint64_t key) {
        a.top_logprobs[(int64_t)row * a.s.top_k + place] = logprob(unordered((uint32_t)(key >> 32)));
        a.top_ids[(int64_t)row * a.s.top_k + place] = (uint32_t)~key;
    };
    join_tops(tops, a.s.slices, a.s.top_k, s_keys[threadIdx.x >> 6], store);
}

}  // namespace

extern "C" {

size_t pw4_token_logprobs_workspace_size(int64_t num_tokens, int64_t vocab, int64_t top_k) {
    if (num_tokens <= 0 || vocab <= 0 || vocab > INT_MAX / 2 || top_k < 0 || top_k > kMaxTop) return 0;
    const int64_t slices = slices_of(num_tokens, vocab);
    return sums_bytes(num_tokens, slices) + (size_t)(num_tokens * slices * top_k) * 8;
}

int pw4_token_logprobs(const void* logits, int dtype, int64_t num_tokens, int64_t vocab, int64_t row_stride,
                       const int64_t* targets, int64_t top_k, float* logprobs, int64_t* ranks, float* entropy,
                       float* top_logprobs, int64_t* top_ids, void* workspace, size_t workspace_bytes,
                       pw4_stream_t stream) {
    if (num_tokens < 0 || vocab <= 0 || top_k < 0) return PW4_ERR_ARG;
    if (dtype != PW4_DTYPE_F16 && dtype != PW4_DTYPE_BF16 && dtype != PW4_DTYPE_F32) return PW4_ERR_ARG;
    if (top_k > kMaxTop || top_k > vocab || vocab > INT_MAX / 2 || num_tokens > 65535 * (int64_t)kThreads ||
        row_stride < vocab) {
        return PW4_ERR_SHAPE;
    }
    if (num_tokens == 0) return PW4_OK;
    if (!logits || !targets || !logprobs || !ranks || !entropy || (top_k && (!top_logprobs || !top_ids))) {
        return PW4_ERR_ARG;
    }
    const size_t element = dtype == PW4_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % element != 0) return PW4_ERR_ARG;
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
        workspace_bytes < pw4_token_logprobs_workspace_size(num_tokens, vocab, top_k)) {
        return PW4_ERR_WORKSPACE;
    }
    const int slices = slices_of(num_tokens, vocab);
    const bool few = per_thread(num_tokens, vocab) == 16;
    const SliceArgs slicing{logits, targets, nullptr, static_cast<SliceSums*>(workspace),
                            reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) + sums_bytes(num_tokens, slices)),
                            row_stride, 0, (int32_t)vocab, (int32_t)top_k, slices, (int32_t)ceil_div(vocab, slices)};
    const LogprobArgs a{slicing, logprobs, ranks, entropy, top_logprobs, top_ids};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    auto run = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        // rows in the grid's second dimension, at most 65535 a launch
        for (int64_t r = 0; r < num_tokens; r += 65535) {
            LogprobArgs part = a;
            const int64_t n = std::min<int64_t>(65535, num_tokens - r);
            part.s.logits = static_cast<const uint8_t*>(logits) + r * row_stride * (int64_t)element;
            part.s.targets = targets + r;
            part.s.sums += r * slices;
            part.s.top += r * slices * top_k;
            part.logprobs += r;
            part.ranks += r;
            part.entropy += r;
            part.top_logprobs += r * top_k;
            part.top_ids += r * top_k;
            part.s.tokens = (int32_t)n;
            if (few) {
                hipLaunchKernelGGL((slice_kernel<DT, 16, true>), dim3(slices, (unsigned)n), dim3(kThreads), 0, s, part.s);
            } else {
                hipLaunchKernelGGL((slice_kernel<DT, 32, true>), dim3(slices, (unsigned)n), dim3(kThreads), 0, s, part.s);
            }
            hipLaunchKernelGGL(join_kernel<DT>, dim3((unsigned)ceil_div(n, kThreads / 64)), dim3(kThreads), 0, s, part);
        }
    };
    if (dtype == PW4_DTYPE_F16) {
        run(std::integral_constant<int, PW4_DTYPE_F16>{});
    } else if (dtype == PW4_DTYPE_BF16) {
        run(std::integral_constant<int, PW4_DTYPE_BF16>{});
    } else {
        run(std::integral_constant<int, PW4_DTYPE_F32>{});
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // extern "C"

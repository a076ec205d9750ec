// Attention of new tokens over a paged cache.
//
// One wave a query and head.  Keys go by in blocks of 64, a key a lane: the lane
// sums q . k_j over its key's row, the block's largest score updates the running
// maximum (running sum and output scaled by e^(old - new)), and the output, four
// elements of the head a lane at most, takes p_j v_j key by key.
#include "pulsar_paged.h"

#include <algorithm>
#include <climits>

#include "paged_common.h"

using namespace pw4;

namespace {

using Args = pw4_paged_attention_args;

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t u) {
    if constexpr (BF16) {
        return __builtin_bit_cast(float, (uint32_t)u << 16);
    } else {
        return (float)__builtin_bit_cast(_Float16, u);
    }
}

template <bool BF16>
__global__ __launch_bounds__(64) void simple_kernel(const Args a) {
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int group = (int)(a.q_heads / a.kv_heads), D = (int)a.head_dim;
    int lo = 0, hi = (int)a.batch;  // the row with cu_q[row] <= t < cu_q[row + 1]
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_q[mid + 1] > t) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    const int b = lo;
    int begin = 0, end = 0;
    if (b < a.batch && t >= a.cu_q[b] && t - a.cu_q[b] < a.max_q_len) {
        const int len = min((int)a.seq_lens[b], (int)a.max_seq_len);
        const int p = a.seq_lens[b] - (a.cu_q[b + 1] - a.cu_q[b]) + (t - a.cu_q[b]);
        end = max(0, min(p + 1, min(len, (int)min((int64_t)INT_MAX, a.table_width * a.page_size))));
        begin = a.window > 0 ? (int)max((int64_t)0, p + 1 - a.window) : 0;
    }
    const int64_t kv_head = (int64_t)(h / group) * a.kv_head_stride;
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + t * a.q_token_stride + h * a.q_head_stride;
    const uint16_t* const kc = static_cast<const uint16_t*>(a.k_cache) + kv_head;
    const uint16_t* const vc = static_cast<const uint16_t*>(a.v_cache) + kv_head;
    float m = -__builtin_inff(), z = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = begin; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        float s = -__builtin_inff();
        int64_t at = 0;
        if (j < end) {
            const int page = a.block_tables[b * a.table_stride + j / a.page_size];
            at = ((uint32_t)page < (uint64_t)a.num_pages ? page : 0) * a.page_stride + j % a.page_size * a.row_stride;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot += to_float<BF16>(q[d]) * to_float<BF16>(kc[at + d]);
            s = dot * a.scale;
            if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float shift = m_new == -__builtin_inff() ? 0.f : m_new;
        const float p = expf(s - shift), scale = expf(m - shift);
        m = m_new;
        z = z * scale + wave_sum(p);
        for (int e = 0; e < 4; ++e) o[e] *= scale;
        for (int k = 0; k < 64 && j0 + k < end; ++k) {
            const float pk = __shfl(p, k);
            const int64_t from = __shfl((long long)at, k);
            for (int e = 0; e < 4; ++e) {
                if (lane + 64 * e < D) o[e] += pk * to_float<BF16>(vc[from + lane + 64 * e]);
            }
        }
    }
    uint16_t* const out = static_cast<uint16_t*>(a.out) + ((int64_t)t * a.q_heads + h) * D;
    for (int e = 0; e < 4; ++e) {
        if (lane + 64 * e < D) out[lane + 64 * e] = f32_to_out<BF16>(z > 0.f ? o[e] / z : z == 0.f ? 0.f : z);
    }
    if (a.lse != nullptr && lane == 0) a.lse[(int64_t)t * a.q_heads + h] = m + logf(z);
}

int check(const Args* a) {
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
    if (!(a->softcap >= 0.f) || a->scale != a->scale) return PW4_ERR_ARG;
    if (a->num_tokens == 0) return PW4_OK;
    if (!a->q || !a->out || !a->cu_q || (a->batch && !a->seq_lens)) return PW4_ERR_ARG;
    if (a->batch && a->table_width && a->num_pages && (!a->k_cache || !a->v_cache || !a->block_tables)) return PW4_ERR_ARG;
    const uint64_t addresses = (uint64_t)(uintptr_t)a->q | (uint64_t)(uintptr_t)a->k_cache |
                               (uint64_t)(uintptr_t)a->v_cache | (uint64_t)(uintptr_t)a->out;
    const uint64_t strides = (uint64_t)(a->q_token_stride | a->q_head_stride | a->page_stride | a->row_stride |
                                        a->kv_head_stride);
    if ((addresses & 15) != 0 || (strides & 7) != 0) return PW4_ERR_ARG;
    return PW4_OK;
}

}  // namespace

extern "C" {

size_t pw4_paged_attention_workspace_size(const pw4_paged_attention_args* args) {
    (void)args;
    return 0;
}

int pw4_paged_attention(const pw4_paged_attention_args* args, void* workspace, size_t workspace_bytes,
                        pw4_stream_t stream) {
    if (const int rc = check(args)) return rc;
    if (args->num_tokens == 0) return PW4_OK;
    (void)workspace;
    (void)workspace_bytes;
    const dim3 grid((unsigned)args->num_tokens, (unsigned)args->q_heads);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (args->dtype == PW4_DTYPE_BF16) {
        hipLaunchKernelGGL(simple_kernel<true>, grid, dim3(64), 0, s, *args);
    } else {
        hipLaunchKernelGGL(simple_kernel<false>, grid, dim3(64), 0, s, *args);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PW4_OK : report_hip_error(e);
}

}  // extern "C"

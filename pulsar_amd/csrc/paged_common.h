// Shared by the paged-cache and log-probability kernels: wave and workgroup
// reductions and scans, and what their C entries need from capi.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "w4a16_common.h"

namespace pw4 {

// Keeps the text for pw4_last_hip_error and returns PW4_ERR_HIP (capi.hip).
int report_hip_error(hipError_t e);
// Compute units of the current device (256 when no device answers).
int device_cus();

// A plan override of the environment (tests and sweeps; null where they are not enabled).
const char* plan_override(const char* name);

constexpr int kWave = 64;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ int wave_inclusive_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    return v;
}

// Inclusive scan over a workgroup of WAVES waves; `total` gets the sum over all
// of them.  Ends with a barrier, so `lds` (WAVES ints) can be used again at once.
template <int WAVES>
__device__ __forceinline__ int block_inclusive_scan(int v, int* lds, int& total) {
    const int wave = threadIdx.x >> 6;
    v = wave_inclusive_scan(v);
    if ((threadIdx.x & 63) == 63) lds[wave] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const int s = lds[w];
        before += w < wave ? s : 0;
        all += s;
    }
    total = all;
    __syncthreads();
    return v + before;
}

}  // namespace pw4

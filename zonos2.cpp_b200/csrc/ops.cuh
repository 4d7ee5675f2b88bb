// ops.cuh — device helpers shared by the device-buffer operators.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

namespace z2b {

// A read-only word: through L1, or past it (`l2`) where a kernel reads ahead of its launch's wait,
// when this SM's L1 may still hold a line of an earlier call.
__device__ __forceinline__ int ld_word(const int* p, bool l2) { return l2 ? __ldcg(p) : *p; }

// The stream that owns packed row t: the last b with row_off[b] <= t, by a 32-way search
// (each round one coalesced-enough load per lane: one round to 32 streams, two to 1024,
// three to OPS_MAX_SEQ). Called by a whole warp; rows ahead of row_off[0] come out as
// stream 0's, so the caller compares t with the stream's first row.
__device__ __forceinline__ int warp_find_seq(const int* row_off, int n_seq, int t, bool l2 = false) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seq;
    while (n > 1) {
        const int step = (n + 31) >> 5;
        const int i = lane * step;
        const bool le = i < n && ld_word(row_off + lo + i, l2) <= t;
        // offsets ascend, so the lanes that hold are a prefix; lane 0 does by construction
        const int c = max(1, __popc(__ballot_sync(0xffffffffu, le)));
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    return lo;
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace z2b

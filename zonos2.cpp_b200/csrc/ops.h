// ops.h — internal interface of the device-buffer operators (include/z2b_ops.h): the
// launches capi_ops.cpp calls after checking the arguments.
#pragma once

#include "../../include/z2b_ops.h"

#include <cuda_runtime.h>

namespace z2b {

// Streams a search over row_off is spread across lanes for, and the prefix_attention plan
// keeps in shared memory.
constexpr int OPS_MAX_SEQ = 4096;

cudaError_t launch_rope_append(const z2b_rope_append_args& a, cudaStream_t s);

// Sizes a prefix_attention call derives from its arguments (host side).
struct AttnPlan;
size_t prefix_attention_bytes(const z2b_prefix_attn_args& a);
// cudaErrorNotSupported when the cache's TMA views cannot be built.
cudaError_t launch_prefix_attention(const z2b_prefix_attn_args& a, cudaStream_t s);

cudaError_t launch_verify(const z2b_verify_args& a, cudaStream_t s);

}  // namespace z2b

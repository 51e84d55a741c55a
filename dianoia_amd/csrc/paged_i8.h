// The attention over an int8 paged cache, for paged_attention.hip's entry point.
#pragma once

#include <hip/hip_runtime.h>

#include "dnx_kernels.h"

namespace dnx {

// Arguments as dnx_paged_attention's, checked there; max_own: the most own keys
// of a sequence that can be seen.
int paged_attention_i8(const dnx_paged_cache* cache, const dnx_paged_batch* batch, const float* q,
                       const float* gate, float* out, int64_t heads, int64_t window,
                       int64_t max_own, hipStream_t stream);

}  // namespace dnx

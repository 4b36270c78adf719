// serve_device.h -- device helpers of the serving operators (serve_kernels.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fl {

typedef _Float16 h16;
typedef __bf16 b16;

// Sequence b's rows [*first, *end) of `total` packed rows.  What the caller wrote into cu is cut to the rows that exist: no start makes a
// kernel leave the buffers.
__device__ inline void seq_rows(const int32_t *cu, int b, int total, int *first, int *end) {
    const int f = min(max(cu[b], 0), total);
    *first = f;
    *end = min(max(cu[b + 1], f), total);
}

}  // namespace fl

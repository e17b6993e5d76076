// The float types that cross the boundary of the 8-bit operators (enum tnns_dtype), one element or one vector at a time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tnns_b200.h"

static inline bool tnns_dtype_ok(int dtype) { return dtype == TNNS_F32 || dtype == TNNS_F16 || dtype == TNNS_BF16; }
static inline int tnns_dtype_bytes(int dtype) { return dtype == TNNS_F32 ? 4 : 2; }

// Runs `...` with T = the type of a checked `dtype`.
#define TNNS_FOR_DTYPE(dtype, T, ...)                       \
    do {                                                    \
        if ((dtype) == TNNS_F32) { using T = float; __VA_ARGS__; } \
        else if ((dtype) == TNNS_F16) { using T = __half; __VA_ARGS__; } \
        else { using T = __nv_bfloat16; __VA_ARGS__; }      \
    } while (0)

#ifdef __CUDACC__
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
}  // namespace
#endif

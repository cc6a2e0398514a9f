// Per-token quantization: one symmetric int8 scale per row, from the row itself.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptq8_ptx.cuh"

namespace ptq8 {

struct RowsParams {
    const void* x;
    int8_t* codes;
    float* scale;
    const int* rows;   // gathered row per output row, or null
    size_t ldx, ldc;   // elements
    long long x_rows;
    int width;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Exact code of y for the 32-bit scale s: round_half_away(y / s).  double(y) / double(s) never
// rounds onto a half-integer that it is not: the quotient of two 24-bit numbers differs from
// k + 1/2 by more than 2^-33 relative, or not at all.
__device__ __forceinline__ int row_code_exact(float y, float s) {
    const double v = static_cast<double>(y) / static_cast<double>(s);
    return static_cast<int>(v >= 0.0 ? floor(v + 0.5) : ceil(v - 0.5));
}

// The simple kernel: one block per row, two passes over the row.
template <typename T>
__global__ void __launch_bounds__(256) rows_kernel(RowsParams p) {
    griddep_launch();
    griddep_wait();
    __shared__ uint32_t part[8];
    const size_t r = blockIdx.x;
    const long long src = p.rows ? p.rows[r] : static_cast<long long>(r);
    int8_t* out = p.codes + r * p.ldc;
    if (src < 0 || src >= p.x_rows) {
        for (int k = threadIdx.x; k < p.width; k += blockDim.x) out[k] = 0;
        if (threadIdx.x == 0) p.scale[r] = 0.0f;
        return;
    }
    const T* x = static_cast<const T*>(p.x) + static_cast<size_t>(src) * p.ldx;
    uint32_t top = 0;   // magnitudes compared as bit patterns: NaN is above infinity is above every number
    for (int k = threadIdx.x; k < p.width; k += blockDim.x) top = max(top, __float_as_uint(to_f32(x[k])) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w) top = max(top, part[w]);
    const float s = top < 0x7F800000u ? fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1e-8f) : __uint_as_float(top);
    for (int k = threadIdx.x; k < p.width; k += blockDim.x)
        out[k] = top < 0x7F800000u ? static_cast<int8_t>(row_code_exact(to_f32(x[k]), s)) : 0;
    if (threadIdx.x == 0) p.scale[r] = s;
}

}  // namespace ptq8

// Products of int8 codes with one scale per token and one per output channel:
//   y[t][c] = fl(fl(float(sum_k x[t][k] w[c][k]) * fl(xs[t] * ws[c])) + b[c]), then the epilogue
// for one weight matrix, or for row groups that each have their own (experts).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptq8_ptx.cuh"

namespace ptq8 {

enum : int { Y_F32 = 0, Y_F16 = 1, Y_BF16 = 2 };

struct LinearParams {
    const int8_t* x;
    const uint8_t* w;
    const float* xs;
    const float* ws;
    const float* bias;       // or null
    void* y;
    const int* offsets;      // or null: one group of all rows
    size_t ldx, ldw, gstride, ldy;
    long long rows;
    int k, n;                // n: output features (channels per gate / up half)
    int groups;
    int y_type;
};

__device__ __forceinline__ void store_y(void* y, size_t at, float v, int type) {
    if (type == Y_F32)
        static_cast<float*>(y)[at] = v;
    else if (type == Y_F16)
        static_cast<__half*>(y)[at] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
}

// Two roundings, then one more for the bias: the engine's dequantization.  A packed int4 code
// stands in the high half of its byte wherever `f` carries the exact factor 1/16.
__device__ __forceinline__ float dequant(int acc, float xs, float ws, float bias) {
    return __fadd_rn(__fmul_rn(__int2float_rn(acc), __fmul_rn(xs, ws)), bias);
}

// silu(g) * u.  exp(-g) overflows to infinity below g = -88, where the quotient is -0.
__device__ __forceinline__ float swiglu(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// Rows of group g, clamped into [0, rows].
__device__ __forceinline__ void group_rows(const LinearParams& p, int g, long long& beg, long long& end) {
    if (!p.offsets) {
        beg = 0;
        end = p.rows;
        return;
    }
    beg = min(max(static_cast<long long>(p.offsets[g]), 0LL), p.rows);
    end = min(max(static_cast<long long>(p.offsets[g + 1]), beg), p.rows);
}

// Up to four bytes that start anywhere, zero past the n-th.
__device__ __forceinline__ uint32_t join4(const uint8_t* p, int n) {
    uint32_t v = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
        if (b < n) v |= static_cast<uint32_t>(p[b]) << (8 * b);
    return v;
}

// The kernel for layouts that neither TMA nor 16-byte loads can read (rows at any byte): 64 tokens x 64 channels
// per block, chunks of 64 codes of both operands joined byte by byte in shared memory, dp4a on 4x4 outputs a
// thread.  The byte loads bound it: 1024 tokens x 1001 -> 1024 takes 72 us, 6.7 us where rows start at
// multiples of 16 bytes (as quantize_rows lays codes, and weights are laid once).
constexpr int kAnyTile = 64;

template <bool W4, bool GATED>
__global__ void __launch_bounds__(256) linear_any_kernel(LinearParams p) {
    constexpr int H = GATED ? 2 : 1, PITCH = 17;   // words per 64-code row, odd against bank conflicts
    __shared__ uint32_t sx[kAnyTile][PITCH], sw[H][kAnyTile][PITCH];
    griddep_launch();
    griddep_wait();
    const int g = blockIdx.z, c0 = blockIdx.x * kAnyTile, tid = threadIdx.x;
    long long beg, end;
    group_rows(p, g, beg, end);
    const int channels = p.n * H;
    const uint8_t* w = p.w + static_cast<size_t>(g) * p.gstride;
    for (long long t0 = beg + static_cast<long long>(blockIdx.y) * kAnyTile; t0 < end;
         t0 += static_cast<long long>(gridDim.y) * kAnyTile) {
        int acc[H][4][4] = {};
        for (int k0 = 0; k0 < p.k; k0 += 64) {
            // a thread joins four codes of one row at a time
            for (int i = tid; i < kAnyTile * 16; i += 256) {
                const int r = i >> 4, k = k0 + (i & 15) * 4;
                uint32_t v = 0;
                if (t0 + r < end) v = join4(reinterpret_cast<const uint8_t*>(p.x) + static_cast<size_t>(t0 + r) * p.ldx + k, p.k - k);
                sx[r][i & 15] = v;
            }
            for (int i = tid; i < H * kAnyTile * 16; i += 256) {
                const int h = i / (kAnyTile * 16), r = (i >> 4) % kAnyTile, k = k0 + (i & 15) * 4, c = c0 + r;
                uint32_t v = 0, rest;
                if (c < p.n) {
                    const uint8_t* row = w + static_cast<size_t>(h * p.n + c) * p.ldw;
                    if (W4)
                        unpack_w4(join4(row + k / 2, min(2, (p.k + 1) / 2 - k / 2)), v, rest);   // x has zeros past its end
                    else
                        v = join4(row + k, p.k - k);
                }
                sw[h][r][i & 15] = v;
            }
            __syncthreads();
#pragma unroll 4
            for (int q = 0; q < 16; ++q) {
                int a[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = static_cast<int>(sx[(tid >> 4) + 16 * i][q]);
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int b = static_cast<int>(sw[h][(tid & 15) + 16 * j][q]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[h][i][j] = __dp4a(a[i], b, acc[h][i][j]);
                    }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long t = t0 + (tid >> 4) + 16 * i;
            if (t >= end) continue;
            const float xs = p.xs[t];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = c0 + (tid & 15) + 16 * j;
                if (c >= p.n) continue;
                float v[H];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const size_t at = static_cast<size_t>(g) * channels + h * p.n + c;
                    v[h] = dequant(acc[h][i][j], xs, p.ws[at], p.bias ? p.bias[at] : 0.0f);
                }
                store_y(p.y, static_cast<size_t>(t) * p.ldy + c, GATED ? swiglu(v[0], v[H - 1]) : v[0], p.y_type);
            }
        }
    }
}

}  // namespace ptq8

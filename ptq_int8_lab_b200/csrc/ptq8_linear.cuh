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

// Two roundings, then one more for the bias: the engine's dequantization.  (Where packed int4 codes are multiplied as
// 16 times the code, `acc` is the sum shifted back: with 1/16 in the scale the product of scales could lose places
// near the smallest normal number.)
__device__ __forceinline__ float dequant(int acc, float xs, float ws, float bias) {
    return __fadd_rn(__fmul_rn(__int2float_rn(acc), __fmul_rn(xs, ws)), bias);
}

// silu(g) * u = g / (1 + exp(-g)) * u.
//
// exp(-g) = 2^t, t = -g log2(e): t's rounding alone would cost |g| units in the last place, so the rest that it leaves
// (exact in one FMA, plus log2(e)'s own rest) goes into the result as 1 + rest * ln 2.  Errors in units of 2^-23:
// exponential 2.5, sum 1/2, reciprocal 1, two products 1/2 each.  (With expf and an IEEE quotient 4096 tokens of 4096 ->
// 2 x 8192 int4 took 272 us instead of 204: the next tile waits for the epilogue's instructions.)
//
// Beyond |g| = 64, which is rare, exp(-g) leaves a float's range before the quotient does (a normal number down to
// g = -91.8), and the rest of an infinite t is not a number.  There, far below zero, the quotient is g exp(g) to the last
// place, exp(g) in two factors: exp(g + 64), the sum exact, and exp(-64).
constexpr float kSiluNear = 64.0f;
constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;

__device__ __forceinline__ float ex2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float silu_far(float g) {
    if (g > 0.0f) return g;   // 1 + exp(-g) is 1
    return g * expf(g + 64.0f) * 1.6038108905486378e-28f;
}
__device__ __forceinline__ float swiglu(float g, float u) {
    if (fabsf(g) > kSiluNear) return silu_far(g) * u;
    const float t = __fmul_rn(g, -kLog2e);
    const float rest = __fmaf_rn(g, kLog2eRest, __fmaf_rn(g, kLog2e, t));   // what t leaves, its sign turned
    const float e = ex2_approx(t);
    const float d = __fmaf_rn(e, __fmul_rn(rest, -kLn2), __fadd_rn(e, 1.0f));
    return __fmul_rn(__fmul_rn(g, rcp_approx(d)), u);
}

// The near steps of swiglu() for two outputs at once.  `most` takes in the denominators: below 2^92 at the end, every gate
// was one that these steps serve (above -63.8; far above zero they give g too).
constexpr float kSwigluMost = 0x1p92f;
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 swiglu2(float2 g, float2 u, float2& most) {
    const float2 t = __fmul2_rn(g, both(-kLog2e));
    const float2 rest = __ffma2_rn(g, both(kLog2eRest), __ffma2_rn(g, both(kLog2e), t));
    const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
    const float2 d = __ffma2_rn(e, __fmul2_rn(rest, both(-kLn2)), __fadd2_rn(e, both(1.0f)));
    most = __fadd2_rn(most, d);
    return __fmul2_rn(__fmul2_rn(g, make_float2(rcp_approx(d.x), rcp_approx(d.y))), u);
}

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
// thread.  The byte loads bound it: 1024 tokens x 1001 -> 1024 takes 90 us, 6.5 us where rows start at
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

// The cache of keys and values in 4 bits: where a token lies, writing rows into it and reading them back.
//
// A row (one token, one head, key or value) is D codes of 4 bits, the even one of a byte low, and a pair of bf16
// (step, least): code c stands for least + step * c.  Pages of a power of two tokens hold the rows of a head one after
// another, so that a tile of keys is one piece of memory.  Step and least are bf16 for its range (half the bytes of
// f32); what their rounding costs stays inside a step, since the codes are computed with the rounded numbers: least is
// rounded down and step up, which keeps 15 steps from least no shorter than the row's spread.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptq8_ptx.cuh"

namespace ptq8 {

struct CacheView {
    uint8_t* k;
    uint8_t* v;
    uint8_t* ks;   // (step, least) pairs, four bytes a row
    uint8_t* vs;
    long long k_page, k_head, v_page, v_head, ks_page, ks_head, vs_page, vs_head;   // bytes
    const int* table;
    long long table_pitch;
    const int* lengths;
    const int* starts;   // or null: one new token per sequence
    long long pages, tokens;
    int width, page, shift, heads, seqs;   // page = 1 << shift tokens
};

// The rows of sequence b among the new tokens, clamped into [0, tokens].
__device__ __forceinline__ void new_rows(const CacheView& c, int b, long long& beg, long long& end) {
    if (!c.starts) {
        beg = b;
        end = b + 1;
        return;
    }
    beg = min(max(static_cast<long long>(c.starts[b]), 0LL), c.tokens);
    end = min(max(static_cast<long long>(c.starts[b + 1]), beg), c.tokens);
}

// The page of position `pos` of sequence b, or -1 where the table has none: behind its end, or not a page.
__device__ __forceinline__ int page_of(const CacheView& c, int b, long long pos) {
    if (pos < 0 || (pos >> c.shift) >= c.width) return -1;
    const int page = c.table[static_cast<long long>(b) * c.table_pitch + (pos >> c.shift)];
    return page >= 0 && page < c.pages ? page : -1;
}

struct CacheRowsParams {
    CacheView c;
    void* k;   // floats [tokens][heads][D]
    void* v;
    long long k_token, k_head, v_token, v_head;   // elements
};

// Eight values of T from (to) memory: as vectors where the rows allow it, one by one otherwise.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2 && __is_same(T, __half)) {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    f[2 * i] = h.x, f[2 * i + 1] = h.y;
                } else {
                    f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b);
template <>
__device__ __forceinline__ uint32_t pair_of<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pair_of<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pair_of<T>(f[0], f[1]), pair_of<T>(f[2], f[3]), pair_of<T>(f[4], f[5]), pair_of<T>(f[6], f[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4)
                p[i] = f[i];
            else if constexpr (__is_same(T, __half))
                p[i] = __float2half_rn(f[i]);
            else
                p[i] = __float2bfloat16_rn(f[i]);
        }
    }
}

// NaN if either is (fminf and fmaxf would drop it).
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Where one row lies: its codes and its pair, or nothing.
struct CacheRow {
    uint8_t* codes = nullptr;
    uint32_t* pair = nullptr;
};

// Row `row` of [tokens][2][heads]: of the keys, then of the values of a token.
template <int D>
__device__ __forceinline__ bool find_row(const CacheRowsParams& p, const int* starts, long long row, long long& token, int& head, bool& value, CacheRow& at) {
    const CacheView& c = p.c;
    token = row / (2 * c.heads);
    const int rest = static_cast<int>(row - token * (2 * c.heads));
    value = rest >= c.heads;
    head = value ? rest - c.heads : rest;
    long long b = token, beg = token, end = token + 1;
    if (c.starts) {
        int lo = 0, hi = c.seqs;   // the last sequence that starts at or before the token
        while (lo + 1 < hi) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= token)
                lo = mid;
            else
                hi = mid;
        }
        b = lo;
        beg = starts[lo];
        end = starts[lo + 1];
        if (beg < 0) beg = 0;
        if (end > c.tokens) end = c.tokens;
        if (token < beg || token >= end) return false;   // of no sequence
    }
    const long long pos = static_cast<long long>(c.lengths[b]) - (end - token);
    const int page = page_of(c, static_cast<int>(b), pos);
    if (page < 0) return true;
    const int in = static_cast<int>(pos & (c.page - 1));
    at.codes = (value ? c.v + page * c.v_page + head * c.v_head : c.k + page * c.k_page + head * c.k_head) + static_cast<long long>(in) * (D / 2);
    at.pair = reinterpret_cast<uint32_t*>(value ? c.vs + page * c.vs_page + head * c.vs_head : c.ks + page * c.ks_page + head * c.ks_head) + in;
    return true;
}

constexpr int kCacheThreads = 256;

// D / 8 lanes a row, eight values a lane:
//   least = the largest bf16 <= min x, step = max(the least bf16 >= fl(fl(max x - least) / 15), 2^-100),
//   code = rint(fl(fl(x - least) * fl(1 / step))) within 0 .. 15.
// A row that holds NaN or an infinity, or whose spread is no finite number, gets codes 0 and NaN for step and least.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheRowsParams p) {
    extern __shared__ int starts[];
    constexpr int LANES = D / 8;
    griddep_wait();
    griddep_launch();
    if (p.c.starts) {
        for (int i = threadIdx.x; i <= p.c.seqs; i += kCacheThreads) starts[i] = p.c.starts[i];
        __syncthreads();
    }
    const int lane = threadIdx.x % LANES;
    const long long rows = p.c.tokens * 2 * p.c.heads, step_rows = static_cast<long long>(gridDim.x) * (kCacheThreads / LANES);
    // a warp's rows go together (the shuffles below take whole warps): rows past the end are not written
    const long long first = (static_cast<long long>(blockIdx.x) * kCacheThreads + threadIdx.x) / LANES;
    const long long warp_first = (static_cast<long long>(blockIdx.x) * kCacheThreads + (threadIdx.x & ~31)) / LANES;
    for (long long row = first, w = warp_first; w < rows; row += step_rows, w += step_rows) {
        long long token = 0;
        int head = 0;
        bool value = false;
        CacheRow at;
        const bool in = row < rows && find_row<D>(p, starts, row, token, head, value, at) && at.codes;
        float f[8] = {};
        if (in) {
            const T* x = value ? static_cast<const T*>(p.v) + token * p.v_token + head * p.v_head : static_cast<const T*>(p.k) + token * p.k_token + head * p.k_head;
            load8<T, VEC>(x + lane * 8, f);
        }
        float lo = f[0], hi = f[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) lo = min_nan(lo, f[i]), hi = max_nan(hi, f[i]);
#pragma unroll
        for (int d = LANES / 2; d; d /= 2) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        if (!in) continue;
        const __nv_bfloat16 least16 = __float2bfloat16_rd(lo);
        const float least = __bfloat162float(least16);
        const __nv_bfloat16 step16 = __float2bfloat16_ru(__fdiv_rn(__fsub_rn(hi, least), 15.0f));
        const float step = fmaxf(__bfloat162float(step16), 0x1p-100f);
        uint32_t codes = 0, pair = 0x7FC07FC0u;   // NaN, NaN
        if (isfinite(least) && isfinite(__bfloat162float(step16))) {
            const float inverse = __frcp_rn(step);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = rintf(__fmul_rn(__fsub_rn(f[i], least), inverse));
                codes |= static_cast<uint32_t>(fminf(fmaxf(q, 0.0f), 15.0f)) << (4 * i);
            }
            pair = (__float_as_uint(step) >> 16) | (__float_as_uint(least) & 0xFFFF0000u);
        }
        reinterpret_cast<uint32_t*>(at.codes)[lane] = codes;
        if (lane == 0) *at.pair = pair;
    }
}

// fl(least + step * code), one rounding to T more.  Positions without a page give zeros.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheRowsParams p) {
    extern __shared__ int starts[];
    constexpr int LANES = D / 8;
    griddep_wait();
    griddep_launch();
    if (p.c.starts) {
        for (int i = threadIdx.x; i <= p.c.seqs; i += kCacheThreads) starts[i] = p.c.starts[i];
        __syncthreads();
    }
    const int lane = threadIdx.x % LANES;
    const long long rows = p.c.tokens * 2 * p.c.heads, step_rows = static_cast<long long>(gridDim.x) * (kCacheThreads / LANES);
    for (long long row = (static_cast<long long>(blockIdx.x) * kCacheThreads + threadIdx.x) / LANES; row < rows; row += step_rows) {
        long long token;
        int head;
        bool value;
        CacheRow at;
        if (!find_row<D>(p, starts, row, token, head, value, at)) continue;
        float f[8] = {};
        if (at.codes) {
            const uint32_t codes = reinterpret_cast<const uint32_t*>(at.codes)[lane], pair = *at.pair;
            const float step = __uint_as_float(pair << 16), least = __uint_as_float(pair & 0xFFFF0000u);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fmaf_rn(step, static_cast<float>((codes >> (4 * i)) & 15), least);
        }
        T* y = value ? static_cast<T*>(p.v) + token * p.v_token + head * p.v_head : static_cast<T*>(p.k) + token * p.k_token + head * p.k_head;
        store8<T, VEC>(y + lane * 8, f);
    }
}

}  // namespace ptq8

// The cache of keys and values in 4 bits: where a token lies, writing rows into it and reading them back.
//
// A row (one token, one head, key or value) is D codes of 4 bits, the even one of a byte low, and a pair of bf16
// (step, least): code c stands for least + step * c.  Pages of a power of two tokens hold the rows of a head one after
// another, so that a tile of keys is one piece of memory.  Step and least are bf16 for its range (half the bytes of
// f32); what their rounding costs stays inside a step, since the codes are computed with the rounded numbers: least is
// rounded down and step up, which keeps 15 steps from least no shorter than the row's spread.
//
// What they spend their time on (in a graph of calls): few rows, a launch after another (32 tokens of 8 heads written and read back 4.1 us);
// many, instructions and what they wait for, at issue 68 %: writing 18 k tokens of 8 heads x 128 (34 us, floor 14) and reading 33 k of 8 x 128
// (40 us, floor 26).
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
    int parts, run;   // warps that share a token's rows, and how many of its steps each has
};

// Eight values of T as they lie in memory: as vectors where the rows allow it, one by one otherwise.
template <typename T, bool VEC>
__device__ __forceinline__ void load8_raw(const T* p, uint32_t (&w)[2 * sizeof(T)]) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = reinterpret_cast<const unsigned short*>(p)[2 * i] | static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[2 * i + 1]) << 16;
    }
}

template <typename T>
__device__ __forceinline__ void values8(const uint32_t (&w)[2 * sizeof(T)], float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (__is_same(T, __half)) {
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = h.x, f[2 * i + 1] = h.y;
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    uint32_t w[2 * sizeof(T)];
    load8_raw<T, VEC>(p, w);
    values8<T>(w, f);
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

// (word & mask) | ones, one instruction.
__device__ __forceinline__ uint32_t mask_or(uint32_t word, uint32_t mask, uint32_t ones) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(word), "r"(mask), "r"(ones));
    return r;
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

// The least and the largest value of a row whose LANES lanes have eight values each; NaN if one is.  f16 and bf16 two at a time,
// the least beside the negative of the largest.
template <typename T>
__device__ __forceinline__ uint32_t least_of(uint32_t a, uint32_t b) {
    if constexpr (__is_same(T, __half)) {
        const __half2 r = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

template <typename T, int LANES>
__device__ __forceinline__ void range_of(const uint32_t (&w)[2 * sizeof(T)], float& lo, float& hi) {
    if constexpr (sizeof(T) == 4) {
        lo = hi = __uint_as_float(w[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) lo = min_nan(lo, __uint_as_float(w[i])), hi = max_nan(hi, __uint_as_float(w[i]));
#pragma unroll
        for (int d = LANES / 2; d; d /= 2) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
    } else {
        constexpr uint32_t kSigns = 0x80008000u;
        const uint32_t a = least_of<T>(least_of<T>(w[0], w[1]), least_of<T>(w[2], w[3]));
        const uint32_t b = least_of<T>(least_of<T>(w[0] ^ kSigns, w[1] ^ kSigns), least_of<T>(w[2] ^ kSigns, w[3] ^ kSigns));
        uint32_t m = least_of<T>(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
        for (int d = LANES / 2; d; d /= 2) m = least_of<T>(m, __shfl_xor_sync(0xffffffffu, m, d));
        if constexpr (__is_same(T, __half)) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
            lo = f.x, hi = -f.y;
        } else {
            lo = __uint_as_float(m << 16), hi = -__uint_as_float(m & 0xFFFF0000u);
        }
    }
}

// Where a new token lies in the cache.
struct CachePlace {
    bool mine;   // it is of a sequence
    int page;    // -1: none
    int in;      // the page
};

__device__ __forceinline__ CachePlace find_token(const CacheView& c, const int* starts, int token) {
    int b = token, end = b + 1;
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
        end = static_cast<int>(min(static_cast<long long>(starts[lo + 1]), c.tokens));
        if (token < max(starts[lo], 0) || token >= end) return {false, -1, 0};
    }
    const long long pos = static_cast<long long>(c.lengths[b]) - (end - token);
    return {true, page_of(c, b, pos), static_cast<int>(pos) & (c.page - 1)};
}

// Row `row` of a token's 2 heads rows, those of the keys first.
struct CacheRow {
    uint8_t* codes;
    uint32_t* pair;
    long long floats;   // its place among k's (v's) elements
    bool value;
};

template <int D>
__device__ __forceinline__ CacheRow row_of(const CacheRowsParams& p, const CachePlace& at, int token, int row) {
    const CacheView& c = p.c;
    const bool value = row >= c.heads;
    const int head = value ? row - c.heads : row;
    uint8_t* codes = (value ? c.v + at.page * c.v_page + head * c.v_head : c.k + at.page * c.k_page + head * c.k_head) + at.in * (D / 2);
    uint8_t* pair = value ? c.vs + at.page * c.vs_page + head * c.vs_head : c.ks + at.page * c.ks_page + head * c.ks_head;
    return {codes, reinterpret_cast<uint32_t*>(pair) + at.in, value ? token * p.v_token + head * p.v_head : token * p.k_token + head * p.k_head, value};
}

constexpr int kCacheThreads = 256;

// D / 8 lanes a row, eight values a lane:
//   least = the largest bf16 <= min x, step = max(the least bf16 >= fl(fl(max x - least) / 15), 2^-100),
//   code = rint(fl(fl(x - least) * fl(1 / step))).
// No code is below 0 or above 15: x >= least, and 15 steps are not shorter than the spread by more than two roundings.  So adding
// 1.5 * 2^23 rounds a quotient to its code, which is then the sum's low bits; the sums' bits, shifted to their places, add
// up to the codes and a constant.  Each operation rounds by itself (no contraction: packed f32 products and sums would be).
// A row that holds NaN or an infinity, or whose spread is no finite number, gets codes 0 and NaN for step and least.
// 291 k rows of 128 bf16 (75 MB in, 20 MB out) in 34 us, issue 68 %.
// U: rows that a lane has at a time.
template <typename T, int D, bool VEC, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheRowsParams p) {
    extern __shared__ int starts[];
    constexpr int LANES = D / 8;
    griddep_wait();
    griddep_launch();
    if (p.c.starts) {
        for (int i = threadIdx.x; i <= p.c.seqs; i += kCacheThreads) starts[i] = p.c.starts[i];
        __syncthreads();
    }
    // a warp has a token's rows, or a part of them: 32 / LANES at a time (the shuffles below take whole warps)
    const int lane = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES, rows = 2 * p.c.heads, steps = (rows + 32 / LANES - 1) / (32 / LANES);
    const unsigned units = static_cast<unsigned>(p.c.tokens) * p.parts;
    for (unsigned unit = (blockIdx.x * kCacheThreads + threadIdx.x) / 32; unit < units; unit += gridDim.x * (kCacheThreads / 32)) {
        const int token = static_cast<int>(unit / static_cast<unsigned>(p.parts)), part = static_cast<int>(unit) - token * p.parts;
        const CachePlace place = find_token(p.c, starts, token);
        if (place.page < 0) continue;
        const int end = min((part + 1) * p.run, steps);
        for (int first = part * p.run; first < end; first += U) {
            CacheRow at[U];
            uint32_t w[U][2 * sizeof(T)];
#pragma unroll
            for (int i = 0; i < U; ++i) {   // (past the end: the last row's again, for the shuffles)
                at[i] = row_of<D>(p, place, token, min(min(first + i, end - 1) * (32 / LANES) + sub, rows - 1));
                load8_raw<T, VEC>(static_cast<const T*>(at[i].value ? p.v : p.k) + at[i].floats + lane * 8, w[i]);
            }
            // lane i % U works out row i's pair and 1 / step
            float lo = 0.0f, hi = 0.0f;
            uint32_t* pair_at = nullptr;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float a, b;
                range_of<T, LANES>(w[i], a, b);
                if (lane % U == i) lo = a, hi = b, pair_at = at[i].pair;
            }
            float least = __bfloat162float(__float2bfloat16_rd(lo));
            const float least_step = __bfloat162float(__float2bfloat16_ru(__fdiv_rn(__fsub_rn(hi, least), 15.0f)));
            const bool good = isfinite(least) && isfinite(least_step);
            const float step = fmaxf(least_step, 0x1p-100f), inverse = good ? __frcp_rn(step) : __int_as_float(0x7FC00000);
            const uint32_t pair = good ? (__float_as_uint(step) >> 16) | (__float_as_uint(least) & 0xFFFF0000u) : 0x7FC07FC0u;   // or NaN, NaN
            if (lane < U && first + lane < end && (first + lane) * (32 / LANES) + sub < rows) *pair_at = pair;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float l = __shfl_sync(0xffffffffu, least, i, LANES), inv = __shfl_sync(0xffffffffu, inverse, i, LANES);
                float f[8];
                values8<T>(w[i], f);
                constexpr float kRound = 0x1.8p23f;
                uint32_t codes = 0, base = 0;
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    codes += __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(f[z], l), inv), kRound)) << (4 * z);
                    base += 0x4B400000u << (4 * z);
                }
                codes = isnan(inv) ? 0 : codes - base;
                if (first + i < end && (first + i) * (32 / LANES) + sub < rows) reinterpret_cast<uint32_t*>(at[i].codes)[lane] = codes;
            }
        }
    }
}

// fl(least + step * code), one rounding to T more.  Positions without a page give zeros.  A code's byte becomes the float 2^23 +
// code by a byte permutation (a conversion runs at a quarter of the rate), and exactly the code by a subtraction.
// 524 k rows of 128 to bf16 (36 MB in, 134 MB out) in 40 us.
// U: rows that a lane has at a time.
template <typename T, int D, bool VEC, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheRowsParams p) {
    extern __shared__ int starts[];
    constexpr int LANES = D / 8;
    griddep_wait();
    griddep_launch();
    if (p.c.starts) {
        for (int i = threadIdx.x; i <= p.c.seqs; i += kCacheThreads) starts[i] = p.c.starts[i];
        __syncthreads();
    }
    const int lane = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES, rows = 2 * p.c.heads, steps = (rows + 32 / LANES - 1) / (32 / LANES);
    const unsigned units = static_cast<unsigned>(p.c.tokens) * p.parts;
    for (unsigned unit = (blockIdx.x * kCacheThreads + threadIdx.x) / 32; unit < units; unit += gridDim.x * (kCacheThreads / 32)) {
        const int token = static_cast<int>(unit / static_cast<unsigned>(p.parts)), part = static_cast<int>(unit) - token * p.parts;
        CachePlace place = find_token(p.c, starts, token);
        if (!place.mine) continue;
        const bool there = place.page >= 0;
        if (!there) place.page = 0;   // (no access to it)
        const int end = min((part + 1) * p.run, steps);
        for (int first = part * p.run; first < end; first += U) {
            CacheRow rows_at[U];
            uint32_t codes[U], pairs[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                rows_at[i] = row_of<D>(p, place, token, min((first + i) * (32 / LANES) + sub, rows - 1));
                codes[i] = there ? reinterpret_cast<const uint32_t*>(rows_at[i].codes)[lane] : 0;
                pairs[i] = there ? *rows_at[i].pair : 0;
            }
#pragma unroll
            for (int i_row = 0; i_row < U; ++i_row) {
                if (first + i_row >= end || (first + i_row) * (32 / LANES) + sub >= rows) continue;
                float f[8];
                const float s = __uint_as_float(pairs[i_row] << 16), l = __uint_as_float(pairs[i_row] & 0xFFFF0000u);
                const uint32_t even = codes[i_row] & 0x0F0F0F0Fu, odd = codes[i_row] >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 c = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7440 + i)), __uint_as_float(__byte_perm(odd, 0x4B000000u, 0x7440 + i))),
                                                make_float2(-0x1p23f, -0x1p23f));
                    const float2 v = __ffma2_rn(make_float2(s, s), c, make_float2(l, l));
                    f[2 * i] = v.x, f[2 * i + 1] = v.y;
                }
                store8<T, VEC>(static_cast<T*>(rows_at[i_row].value ? p.v : p.k) + rows_at[i_row].floats + lane * 8, f);
            }
        }
    }
}

}  // namespace ptq8

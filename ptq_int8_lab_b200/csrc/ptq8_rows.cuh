// Per-token quantization: one symmetric int8 scale per row, from the row itself.
//
// One read, one write: 8192 x 4096 bf16 in 17.3 us (100.7 MB at 5.8 TB/s, 90 % of a plain copy), f32 in 25.7 us
// (98 %).  Instructions come next (11 M warp instructions for the former, issue slots 70 % busy): they bound
// the gathered form, which reads a token from L2 once per row that asks for it (16384 rows of 2048 f16 15.7 us).
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
    long long x_rows, n_rows;
    int width;
};

// How one 16-byte vector of T is read: its largest magnitude as a 32-bit pattern (NaN above infinity
// above every number, so a maximum of patterns loses neither), and its values.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ uint32_t join(uint32_t m, uint32_t w) { return max(m, w & 0x7FFFFFFFu); }
    static __device__ __forceinline__ uint32_t top(uint32_t m) { return m; }
    static __device__ __forceinline__ void values(const uint4& v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ uint32_t join(uint32_t m, uint32_t w) {
        const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&m), __habs2(*reinterpret_cast<__nv_bfloat162*>(&w)));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t top(uint32_t m) { return max(m & 0xFFFFu, m >> 16) << 16; }
    static __device__ __forceinline__ void values(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <>
struct Vec<__half> {
    static constexpr int V = 8;
    static __device__ __forceinline__ uint32_t join(uint32_t m, uint32_t w) {
        const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&m), __habs2(*reinterpret_cast<__half2*>(&w)));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t top(uint32_t m) {
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m & 0xFFFFu, m >> 16)))));
    }
    static __device__ __forceinline__ void values(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
};

__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The first n (>= 1) elements of a vector one by one; the others are zero (code 0, no part in the maximum).
template <typename T>
__device__ __noinline__ uint4 load_part(const T* p, int n) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < Vec<T>::V; ++i) {
        if (i < n) {
            if (sizeof(T) == 4)
                w[i] = reinterpret_cast<const uint32_t*>(p)[i];
            else
                w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[i]) << (16 * (i & 1));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The first n elements of a vector, zero in the others' place.
template <typename T>
__device__ __forceinline__ uint4 first_of(uint4 q, int n) {
    if (n >= Vec<T>::V) return q;
    uint32_t* w = &q.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int here = (n * static_cast<int>(sizeof(T)) - 4 * i);   // bytes of this word that count
        w[i] = here >= 4 ? w[i] : here <= 0 ? 0u : w[i] & 0xFFFFu;
    }
    return q;
}

// A whole vector that starts `off` bytes past a multiple of 16 (off: the same for a row's vectors, so for a
// warp): two aligned loads joined.  Both lie inside the tensor, or the caller loads one by one.
__device__ __forceinline__ uint4 load_shifted(const void* p, uint32_t off) {
    const char* a = static_cast<const char*>(p) - off;
    const uint4 x = load16(a);
    if (off == 0) return x;
    const uint4 y = load16(a + 16);
    const uint32_t bits = (off & 3) * 8;
    switch (off >> 2) {
        case 0: return make_uint4(__funnelshift_r(x.x, x.y, bits), __funnelshift_r(x.y, x.z, bits), __funnelshift_r(x.z, x.w, bits), __funnelshift_r(x.w, y.x, bits));
        case 1: return make_uint4(__funnelshift_r(x.y, x.z, bits), __funnelshift_r(x.z, x.w, bits), __funnelshift_r(x.w, y.x, bits), __funnelshift_r(y.x, y.y, bits));
        case 2: return make_uint4(__funnelshift_r(x.z, x.w, bits), __funnelshift_r(x.w, y.x, bits), __funnelshift_r(y.x, y.y, bits), __funnelshift_r(y.y, y.z, bits));
        default: return make_uint4(__funnelshift_r(x.w, y.x, bits), __funnelshift_r(y.x, y.y, bits), __funnelshift_r(y.y, y.z, bits), __funnelshift_r(y.z, y.w, bits));
    }
}

// Codes of one vector: round_half_away(f / s), the exact quotient.  Multipliers that bracket 1/s, each in
// one FMA with 1.5 * 2^23 added: the sum lies in [2^23, 2^24) where floats are 1 apart, so it is rounded to
// the nearest integer and its low byte is the code (|f / s| <= 127 (1 + 2^-23): s is the row's own).  Where
// both agree, every number between f * inv_lo and f * inv_hi rounds to that integer, and so does the exact
// quotient, which lies strictly inside.  Where they do not (`flag`), a half-integer t lies between them, and
// the sign of f - t s decides: one FMA, whose rounding keeps the sign of the exact value.
// The first n < 8 codes of a vector, in the largest pieces that their place allows.
__device__ __forceinline__ void store_first(int8_t* out, uint2 c, int n, bool words) {
    if (words) {   // out is a multiple of the vector's codes
        if (n & 4) *reinterpret_cast<uint32_t*>(out) = c.x;
        const uint32_t rest = n & 4 ? c.y : c.x;
        out += n & 4;
        if (n & 2) *reinterpret_cast<unsigned short*>(out) = static_cast<unsigned short>(rest);
        if (n & 1) out[n & 2] = static_cast<int8_t>(rest >> (n & 2 ? 16 : 0));
        return;
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) out[i] = static_cast<int8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
}

constexpr float kRowMagic = 12582912.0f;

template <int V>
__device__ __forceinline__ void pack_codes(const uint32_t (&m)[V], uint32_t (&out)[V / 4]) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k)
        out[k] = __byte_perm(__byte_perm(m[4 * k], m[4 * k + 1], 0x0040), __byte_perm(m[4 * k + 2], m[4 * k + 3], 0x0040), 0x5410);
}

template <int V>
__device__ __forceinline__ void codes_of(const float (&f)[V], float inv_lo, float inv_hi, uint32_t (&out)[V / 4], uint32_t& flag) {
    const float2 lo = make_float2(inv_lo, inv_lo), hi = make_float2(inv_hi, inv_hi), mg = make_float2(kRowMagic, kRowMagic);
    uint32_t m[V];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        const float2 y = make_float2(f[i], f[i + 1]);
        const float2 a = __ffma2_rn(y, lo, mg), b = __ffma2_rn(y, hi, mg);
        flag |= __float_as_uint(a.x) ^ __float_as_uint(b.x);
        flag |= __float_as_uint(a.y) ^ __float_as_uint(b.y);
        m[i] = __float_as_uint(a.x);
        m[i + 1] = __float_as_uint(a.y);
    }
    pack_codes<V>(m, out);
}

template <int V>
__device__ __forceinline__ void codes_exact(const float (&f)[V], float inv_lo, float inv_hi, float s, uint32_t (&out)[V / 4]) {
    uint32_t m[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float a = __fmaf_rn(f[i], inv_lo, kRowMagic) - kRowMagic, b = __fmaf_rn(f[i], inv_hi, kRowMagic) - kRowMagic;
        const float k = fminf(a, b), d = __fmaf_rn(-(k + 0.5f), s, f[i]);
        m[i] = __float_as_uint((a == b ? a : (d > 0.0f || (d == 0.0f && f[i] > 0.0f)) ? k + 1.0f : k) + kRowMagic);
    }
    pack_codes<V>(m, out);
}

// One pass over the data: TPR threads per row hold it in registers, NV vectors of 16 bytes each,
// between its maximum and its codes.  (NV 0, for rows longer than that: a loop that reads them twice.)
// PLAIN: rows of whole vectors that start at multiples of 16 bytes, codes that can be stored in words.
// Instructions bound it, not memory, so that the common form has no other case in it.
template <typename T, int TPR, int NV, bool PLAIN>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) rows_kernel(RowsParams p) {
    constexpr int V = Vec<T>::V, kBlock = TPR > 128 ? TPR : 128, kWarps = TPR / 32, kHeld = NV ? NV : 1;
    __shared__ uint32_t part[kBlock / 32];
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x % TPR;
    const size_t r = static_cast<size_t>(blockIdx.x) * (kBlock / TPR) + threadIdx.x / TPR;
    const bool there = r < static_cast<size_t>(p.n_rows);
    const long long src = !there ? -1 : p.rows ? p.rows[r] : static_cast<long long>(r);
    const bool read = src >= 0 && src < p.x_rows;
    const T* x = static_cast<const T*>(p.x) + static_cast<size_t>(read ? src : 0) * p.ldx;
    // Not PLAIN: where the row starts, and whether aligned loads around its vectors stay inside the tensor (they
    // may leave it in its first and last row).
    const uint32_t off = PLAIN ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 15);
    const bool inner = PLAIN || (src > 0 && src + 1 < p.x_rows && p.ldx >= 16);
    const int vecs = (p.width + V - 1) / V, readable = read ? vecs : 0;
    auto fetch = [&](int v) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (v < readable) {
            if (PLAIN)
                q = load16(x + v * V);
            else if (inner)
                q = first_of<T>(load_shifted(x + v * V, off), p.width - v * V);
            else
                q = load_part(x + v * V, min(V, p.width - v * V));
        }
        return q;
    };
    uint32_t top = 0;
    auto join = [&](const uint4& q) { top = Vec<T>::join(Vec<T>::join(Vec<T>::join(Vec<T>::join(top, q.x), q.y), q.z), q.w); };
    uint4 d[kHeld];
    if (NV) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) d[i] = fetch(lane + i * TPR);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) join(d[i]);
    } else {
        for (int v = lane; v < vecs; v += TPR) join(fetch(v));
    }
    top = __reduce_max_sync(0xffffffffu, Vec<T>::top(top));
    if (kWarps > 1) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
        const int w0 = threadIdx.x / TPR * kWarps;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = max(top, part[w0 + w]);
    }
    if (!there) return;
    const bool finite = top < 0x7F800000u;
    float s = __uint_as_float(top), inv_lo = 0.0f, inv_hi = 0.0f;   // not finite: codes 0
    if (finite) {
        s = fmaxf(__fdiv_rn(s, 127.0f), 1e-8f);
        // 1/s within half a unit, then at least 2^-23 relative to both sides
        const float inv = __frcp_rn(s);
        inv_lo = __fmul_rd(inv, 1.0f - 0x1p-22f);
        inv_hi = __fmul_ru(inv, 1.0f + 0x1p-22f);
    }
    if (lane == 0) p.scale[r] = read ? s : 0.0f;
    int8_t* out = p.codes + r * p.ldc;
    const bool words = PLAIN || (reinterpret_cast<uintptr_t>(out) & (V - 1)) == 0;
    auto emit = [&](int v, const uint4& q) {
        if (v >= vecs) return;
        float f[V];
        uint32_t c[V / 4], flag = 0;
        Vec<T>::values(q, f);
        codes_of<V>(f, inv_lo, inv_hi, c, flag);
        if (flag) codes_exact<V>(f, inv_lo, inv_hi, s, c);
        if (!finite) c[0] = c[V / 4 - 1] = 0;
        if (PLAIN || (words && (v + 1) * V <= p.width)) {
            if (V == 8)
                *reinterpret_cast<uint2*>(out + v * V) = make_uint2(c[0], c[V / 4 - 1]);
            else
                *reinterpret_cast<uint32_t*>(out + v * V) = c[0];
        } else {
            store_first(out + v * V, make_uint2(c[0], c[V / 4 - 1]), min(V, p.width - v * V), words);
        }
    };
    if (NV) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) emit(lane + i * TPR, d[i]);
    } else {
        for (int v = lane; v < vecs; v += TPR) emit(v, fetch(v));
    }
}

}  // namespace ptq8

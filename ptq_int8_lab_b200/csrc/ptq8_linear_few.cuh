// The product for a few tokens: dp4a on weights that go from memory straight to registers.
//
// One or a few tokens cannot fill a tensor-core tile, and the tile's way (shared memory, TMEM, barriers,
// partial sums between CTAs) costs more than the arithmetic.  Here a warp owns four weight rows (gated: two
// gate and two up rows), a lane 16 bytes of each at a time, and the only exchange is the warp's sum at the
// end.  Where rows are few and long, KS warps of a block share four rows' input features.
//
// Bound by the weights' way from DRAM and the launch: one token x 4096 x 4096 takes 5.2 us (int4 4.0 us) with
// weights from DRAM, 3.8 us (3.6 us) from L2; 1024 x 1024 takes 2.0 us, of which a launch after another is 1.3.
#pragma once

#include "ptq8_linear.cuh"

namespace ptq8 {

constexpr int kFewWarps = 8, kFewRows = 4;

struct FewParams {
    LinearParams l;
    int ks;   // warps that share four rows' sum: a power of two
};

// Plain loads, not read-only ones: with programmatic launch the tensors may be written while this kernel has started.
__device__ __forceinline__ uint4 ld16(const void* p) { return *static_cast<const uint4*>(p); }

// acc += the products of 4 words of weights with 4 words of codes.
__device__ __forceinline__ int dot16(const uint4& w, const uint4& x, int acc) {
    acc = __dp4a(static_cast<int>(w.x), static_cast<int>(x.x), acc);
    acc = __dp4a(static_cast<int>(w.y), static_cast<int>(x.y), acc);
    acc = __dp4a(static_cast<int>(w.z), static_cast<int>(x.z), acc);
    return __dp4a(static_cast<int>(w.w), static_cast<int>(x.w), acc);
}

// A lane's codes of one token for 16 bytes of weights.  int4: 32 codes, those at even places and those at
// odd places apart, as the halves of the weights' bytes are.
template <bool W4>
struct FewCodes {
    uint4 even, odd;
};
template <bool W4>
__device__ __forceinline__ FewCodes<W4> few_codes(const uint4& a, const uint4& b) {
    FewCodes<W4> c;
    if (W4) {
        c.even = make_uint4(__byte_perm(a.x, a.y, 0x6420), __byte_perm(a.z, a.w, 0x6420), __byte_perm(b.x, b.y, 0x6420),
                            __byte_perm(b.z, b.w, 0x6420));
        c.odd = make_uint4(__byte_perm(a.x, a.y, 0x7531), __byte_perm(a.z, a.w, 0x7531), __byte_perm(b.x, b.y, 0x7531),
                           __byte_perm(b.z, b.w, 0x7531));
    } else {
        c.even = c.odd = a;
    }
    return c;
}
template <bool W4>
__device__ __forceinline__ int few_dot(const uint4& w, const FewCodes<W4>& c, int acc) {
    if (!W4) return dot16(w, c.even, acc);
    // 16 times each code, in its byte's high half (the sum is shifted back)
    const uint32_t m = 0xF0F0F0F0u;
    acc = dot16(make_uint4((w.x << 4) & m, (w.y << 4) & m, (w.z << 4) & m, (w.w << 4) & m), c.even, acc);
    return dot16(make_uint4(w.x & m, w.y & m, w.z & m, w.w & m), c.odd, acc);
}

// MT tokens at a time; a group's further rows read its weights again (from L2).
template <int MT, bool W4, bool GATED>
__global__ void __launch_bounds__(32 * kFewWarps, MT == 4 ? 2 : 4) linear_few_kernel(FewParams p) {
    constexpr int H = GATED ? 2 : 1, C = kFewRows / H;   // channels of a warp
    __shared__ int sums[kFewWarps][kFewRows * MT];
    const LinearParams& l = p.l;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = warp & (p.ks - 1), set = warp / p.ks;
    const int c0 = (blockIdx.x * (kFewWarps / p.ks) + set) * C;   // first channel of this warp
    const int bytes = W4 ? l.k / 2 : l.k;   // whole vectors of 16 (the host sees to it)
    const int g = blockIdx.y;
    const uint8_t* w = l.w + static_cast<size_t>(g) * l.gstride;
    const uint8_t* row[kFewRows];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r)   // rows past the end repeat the last one; their sums are dropped
        row[r] = w + (static_cast<size_t>(r / C) * l.n + min(c0 + r % C, l.n - 1)) * l.ldw;
    // this warp's share of the row: whole strides of 512 bytes
    const int strides = (bytes + 511) / 512, s0 = strides * part / p.ks, s1 = strides * (part + 1) / p.ks;
    griddep_launch();
    if (!l.offsets) {   // into L2 while the kernel before this one drains
        const int n = min(s1 * 512, bytes) - s0 * 512;
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
            if (lane == r && n > 0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row[r] + s0 * 512), "r"(n) : "memory");
    }
    griddep_wait();
    long long beg, end;
    group_rows(l, g, beg, end);
    // the lane's output: row r, token t of the pass; its scales are loaded ahead of the sums
    const int r_lane = lane / MT, t_lane = lane % MT, c = c0 + r_lane % C;
    const bool mine_ok = part == 0 && lane < kFewRows * MT && c < l.n && beg < end;
    const size_t at = static_cast<size_t>(g) * (l.n * H) + (r_lane / C) * l.n + c;
    const float ws = mine_ok ? l.ws[at] : 0.0f;
    const float bias = mine_ok && l.bias ? l.bias[at] : 0.0f;
    for (long long t0 = beg; t0 < end; t0 += MT) {
        const int tokens = static_cast<int>(min(static_cast<long long>(MT), end - t0));
        const bool here = mine_ok && t_lane < tokens;
        const float xs = here ? l.xs[t0 + t_lane] : 0.0f;
        int acc[kFewRows][MT] = {};
        const uint8_t* x[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t)   // missing tokens repeat the last one; their sums are dropped
            x[t] = reinterpret_cast<const uint8_t*>(l.x) + static_cast<size_t>(t0 + min(t, tokens - 1)) * l.ldx;
        const int whole = min(s1, bytes / 512);   // strides that every lane has a part of
#pragma unroll 2
        for (int s = s0; s < whole; ++s) {
            const int k = s * 512 + lane * 16;
            uint4 wv[kFewRows];
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) wv[r] = ld16(row[r] + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const FewCodes<W4> c = W4 ? few_codes<W4>(ld16(x[t] + 2 * k), ld16(x[t] + 2 * k + 16)) : few_codes<W4>(ld16(x[t] + k), wv[0]);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) acc[r][t] = few_dot<W4>(wv[r], c, acc[r][t]);
            }
        }
        if (max(s0, whole) < s1) {   // the row's last stride, of whole vectors
            const int k = max(s0, whole) * 512 + lane * 16;
            const uint4 zero = make_uint4(0, 0, 0, 0);
            const bool in = k < bytes;
            uint4 wv[kFewRows];
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) wv[r] = in ? ld16(row[r] + k) : zero;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const FewCodes<W4> c = few_codes<W4>(in ? ld16(x[t] + (W4 ? 2 * k : k)) : zero, in && W4 ? ld16(x[t] + 2 * k + 16) : zero);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) acc[r][t] = few_dot<W4>(wv[r], c, acc[r][t]);
            }
        }
        // lane i keeps the warp's sum of row i / MT, token i % MT
        int mine = 0;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int sum = __reduce_add_sync(0xffffffffu, acc[r][t]);
                if (lane == r * MT + t) mine = sum;
            }
        if (p.ks > 1) {
            if (lane < kFewRows * MT) sums[warp][lane] = mine;
            __syncthreads();
            if (part == 0 && lane < kFewRows * MT)
                for (int i = 1; i < p.ks; ++i) mine += sums[warp + i][lane];
        }
        float v = here ? dequant(W4 ? mine >> 4 : mine, xs, ws, bias) : 0.0f;
        if (GATED) v = swiglu(v, __shfl_down_sync(0xffffffffu, v, C * MT));
        if (here && r_lane < C) store_y(l.y, static_cast<size_t>(t0 + t_lane) * l.ldy + c, v, l.y_type);
        if (p.ks > 1) __syncthreads();
    }
}

}  // namespace ptq8

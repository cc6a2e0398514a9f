// Attention over the cache of 4-bit keys and values.
//
// A code enters the tensor cores as a normal f16 number around zero (16 times it, for the second code of a byte): masked out of a word
// together with the exponent of 1024, less 1032.  Nine instructions widen eight codes; the steps and the middles go into the numbers
// around the products:
//   q . key    = step_k (q . (codes - 8)) + (least_k + 8 step_k) sum(q)       queries as f16 times a power of two
//   sum p v    = sum (p step_v) (codes - 8) + sum p (least_v + 8 step_v)      p step_v as f16, over a bound of step_v
// A query is scaled by the power of two that takes its largest value to 2^14 .. 2^15, dimensions that meet a byte's second code to
// a sixteenth of that: what is within 2^28 (2^24) of the largest keeps f16's and bf16's places.  p step_v is rounded to f16's 11 bits (an
// output has 11, or bf16's 8), with 2^-24 of the largest as its finest step; everything else is f32.
// (The four bits alone are, read as f16, the subnormal number code * 2^-24: five instructions for eight codes.  But terms that do not all
// have one sign lose less to p's rounding, and the tensor cores, which line the products of a sum up by their operands' exponents and
// cut what is below, take a subnormal number's exponent for 2^-14.  131072 f16 tokens, which average to 0.4 % of a value: 7.5e-4 from 64
// bits with such codes of values, 2.7e-4 like this; the output's own rounding is 2.1e-4.  One dimension of queries 2^12 times the
// others, where keys are zero: 4e-3 with such codes of keys.)
//
// A warp takes 16 tokens as the rows of its products, 8 NT query rows (query token x head of a key's group) as
// the columns: keys codes [16 tokens x D] x queries [D x rows], then values codes [D x 16 tokens] x p [16 tokens x rows].
// Which of a lane's codes stands for which place of a product is free as long as both operands agree, so a lane reads
// its keys and values from the cache's own order, 4 D / 32 and 4 D / 64 words at a time.
//
// The softmax is kept running: a row's reference is moved only when a score passes it by 8 (in powers of two), a vote of
// the warp that fails almost always, and the sums of 8 lanes meet at the end of a segment.
//
// Work is units of 128 tokens of one key head and row tile.  All sequences' units lie in one order, and CTA c of N takes
// those from c U / N to (c + 1) U / N: equal shares whatever the lengths are, known on the device only.  A row tile cut
// by a share's end leaves (numerators, reference, sum) in the workspace, and a second kernel joins them.
//
// What it spends its time on: for few rows the way from one launch to the next (one token over 2000 positions 9.2 us, of which the join's
// launch and set-up are half), then the loop and the ends (32 sequences of up to 8192 tokens 30 us, floor 12, issue 56 %: 3 us to the first
// bytes, shares that end apart, the join 6); warp-level products reach 42 % of their rate with 8 computing warps an SM.  All variants
// spill a little (48 to 166 bytes of stores), 64 dimensions with 8 rows aside.
// A producer warp keeps bulk copies of whole tiles in flight; four warps compute, RW of them on different rows, 4 / RW on
// different tokens of a tile.
#pragma once

#include "ptq8_cache.cuh"
#include "ptq8_linear.cuh"

namespace ptq8 {

constexpr int kAttTile = 128, kAttWarps = 4, kAttThreads = 32 * (kAttWarps + 1);
constexpr float kAttNone = -0x1.fffffep127f;   // reference of a row that has seen nothing: no score is less
constexpr float kAttSlack = 8.0f;
// What a row tile costs beside its tokens (queries in, numerators joined and out), in units.
constexpr int kAttOver = 2;
// Units at most, which the host sees to; starts that decrease (their tokens count for several sequences) are held to it on the device.
constexpr int kAttUnits = 0x3FFFFFFF;

struct AttDesc {
    int first, last;       // the CTAs that have parts of a row tile that is cut (last -1: it is not)
    int rows, head, row0;  // of the sequence; the tile's key head and first row
    int token0;            // of its sequence
    int pad[2];
};

struct AttParams {
    CacheView c;
    const void* q;
    void* out;
    long long q_token, q_head, o_token, o_head;   // elements
    // scale * log2(e) = 2^kAttKeys key_scale * score_scale, a power of two: products of scores with that are exact, so that a row's largest score
    // becomes its reference exactly, however large it is
    float key_scale, score_scale;
    int per;            // query heads of a key head
    int by_item;        // 1: a CTA per row tile, none cut; 0: equal shares
    int listed;         // descriptions by row tile (one new token per sequence, no more row tiles than CTAs), not by CTA
    int type;           // Y_F16 or Y_BF16
    int vec_q, vec_o;   // rows at multiples of 16 bytes
    float* part;        // [2 N][R][D] numerators
    float* stat;        // [2 N][R][2] reference, sum
    AttDesc* desc;      // [N], or by row tile
    long long wait_limit;
    int* err;
    int stall;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values, transposed: lane i's pair (row i / 4, columns 2 (i % 4) ..) becomes (column, rows).
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&w)[W], const uint8_t* p) {
    if constexpr (W == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
    }
}

// 2^e for e within -126 .. 127.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// 2^e takes a query's largest value to 2^14 .. 2^15 (below 2^-112 it stays below, as subnormal numbers do).
__device__ __forceinline__ int att_power(float top) { return min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126); }

// Keys are multiplied by 2^-kAttKeys (in key_scale), so that neither what takes a product back to its size, 2^(kAttKeys - e), leaves f32's
// range for any query, nor products with queries of 2^14 do for keys up to 2^115.
constexpr int kAttKeys = 13;

// a / b of powers of two within 2^+-121, 2^-126 at least.
__device__ __forceinline__ float power_ratio(float a, float b) {
    return exp2_int(max((__float_as_int(a) >> 23) - (__float_as_int(b) >> 23), -126));
}

template <int D, int NT, int RW>
struct AttShape {
    static constexpr int R = 8 * NT * RW, TW = kAttWarps / RW;
    static constexpr int H = 2;   // products of 16 tokens at a time
    static constexpr int kPerSm = D * NT <= 128 ? 3 : 2;
    static constexpr int kStages = D == 256 ? 2 : 3;
    static constexpr int kCodes = kAttTile * D / 2, kPairs = kAttTile * 4, kStage = 2 * (kCodes + kPairs);
    static constexpr int kPitch = D + 4;   // floats of a row of the joining buffer, off the banks' period
    static constexpr int kJoin = kAttWarps * 8 * NT * kPitch * 4, kStats = kAttWarps * 8 * NT * 2 * 4;
    // a warp's query fragments lie in its own part of the joining buffer, which it writes when it is done with them
    static constexpr int kWarp = 8 * NT * kPitch * 4;
    static_assert(NT * (D / 32) * 32 * 16 + NT * 32 * 8 <= kWarp && kJoin == kAttWarps * kWarp, "query fragments and the rows' c fit");
    // query rows that the producer fetches ahead (the largest tile of 256 dimensions has no room for them)
    static constexpr bool kAhead = D < 256 || RW < 4;
    static constexpr int kQueries = kAhead ? R * D * 2 : 0;
    static constexpr int smem(int seqs) { return kStages * kStage + kJoin + kQueries + kStats + (seqs + 1) * 4; }
    static_assert(kPerSm * (smem(1024) + 1024 + 256) <= 228 * 1024, "shared memory of an SM");
};

// A warp's query rows and what it has of their softmax.  Lane (g, t) = (lane / 4, lane % 4) holds, for the products,
// row g of each tile of 8; of the sums, rows 2 t and 2 t + 1.
template <int D, int NT>
struct AttRows {
    const uint4* q;               // fragments [NT][D / 32][32 lanes]: of a word of keys, those of its codes 0, 4; 1, 5; 2, 6; 3, 7
    float2 a[NT], b[NT];          // score in powers of two = a * (step (q . (codes - 8)) + middle b), step and middle times key_scale; a: a power of two
    float2 m[NT], l[NT], lo[NT];  // reference, sum of p, sum of p (least_v + 8 step_v)
    int lim[NT][2];               // positions that the row sees
    float o[D / 16][NT][4];
    float c;                             // what p step_v is multiplied by: a power of two, by the steps of the values that a row sees
    bool apart;                          // the rows' c differ and lie behind q ([NT][32 lanes], of rows 2 t and 2 t + 1): MASKED steps from here on
    __device__ __forceinline__ float2* own_c() const {
        return reinterpret_cast<float2*>(const_cast<uint4*>(q - (threadIdx.x & 31)) + NT * (D / 32) * 32) + (threadIdx.x & 31);
    }
    __device__ __forceinline__ float2 c_of(int nt) const { return apart ? own_c()[nt * 32] : make_float2(c, c); }
};

__device__ __forceinline__ float att_value(const void* p, long long at, int type) {
    return type == Y_F16 ? __half2float(static_cast<const __half*>(p)[at]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

// The lane's part of the query rows from `row0` on: D / 4 values of each tile's row g.  ahead: those rows in shared memory, or null.
template <int D, int NT>
__device__ __forceinline__ void att_queries(const AttParams& p, AttRows<D, NT>& r, uint4* q, long long token0, int n, int head, int row0, int rows, long long len, const void* ahead) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int DL = D / 4;
    const long long cap = static_cast<long long>(p.c.width) << p.c.shift;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + g;
        float f[DL];
        if (row < rows) {
            const int i = row / p.per, j = row - i * p.per;
            const long long at = (token0 + i) * p.q_token + static_cast<long long>(head * p.per + j) * p.q_head + t * DL;
            if (p.vec_q) {
                const char* from = ahead ? static_cast<const char*>(ahead) + ((nt * 8 + g) * D + t * DL) * 2 : static_cast<const char*>(p.q) + 2 * at;
#pragma unroll
                for (int k = 0; k < DL / 8; ++k) {
                    float e[8];
                    if (p.type == Y_F16)
                        load8<__half, true>(reinterpret_cast<const __half*>(from) + 8 * k, e);
                    else
                        load8<__nv_bfloat16, true>(reinterpret_cast<const __nv_bfloat16*>(from) + 8 * k, e);
#pragma unroll
                    for (int z = 0; z < 8; ++z) f[8 * k + z] = e[z];
                }
            } else {
#pragma unroll
                for (int k = 0; k < DL; ++k) f[k] = att_value(p.q, at + k, p.type);
            }
        } else {
#pragma unroll
            for (int k = 0; k < DL; ++k) f[k] = 0.0f;
        }
        float top = 0.0f, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < DL; ++k) top = max_nan(top, fabsf(f[k]));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = att_power(top);
        const float up = exp2_int(e);
#pragma unroll
        for (int k = 0; k < DL; ++k) {
            f[k] *= up;
            sum += f[k];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // codes 0, 4 of a word in one register, 1, 5 (which come 16 times too large), 2, 6 and 3, 7
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
            const float* x = f + 8 * w;
            q[(nt * (D / 32) + w) * 32 + lane] = make_uint4(pair_of<__half>(x[0], x[4]), pair_of<__half>(x[1] * 0.0625f, x[5] * 0.0625f),
                                                            pair_of<__half>(x[2], x[6]), pair_of<__half>(x[3] * 0.0625f, x[7] * 0.0625f));
        }
        // the products are 2^e of the true ones, keys 2^-kAttKeys; NaN and infinities in a row make all of its scores NaN
        const float a = isfinite(top) ? exp2_int(kAttKeys - e) * p.score_scale : __int_as_float(0x7FC00000);
        const float b = sum;
        r.a[nt] = make_float2(__shfl_sync(0xffffffffu, a, 8 * t), __shfl_sync(0xffffffffu, a, 8 * t + 4));
        r.b[nt] = make_float2(__shfl_sync(0xffffffffu, b, 8 * t), __shfl_sync(0xffffffffu, b, 8 * t + 4));
        r.m[nt] = both(kAttNone);
        r.l[nt] = r.lo[nt] = both(0.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int my = row0 + nt * 8 + 2 * t + i;
            // query i of n sees the positions up to its own; rows past the end see all (nothing is kept of them)
            r.lim[nt][i] = my < rows ? static_cast<int>(min(max(len - n + my / p.per + 1, 0LL), cap)) : 0x7FFFFFFF;
        }
    }
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) r.o[mt][nt][i] = 0.0f;
    r.c = 0x1p120f;   // as for a bound of 2^-113 on step_v
    r.apart = false;
    r.q = q + lane;
    __syncwarp();
}

constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;

// Codes less eight (16 times that for the high one of a byte) as normal f16 numbers: 1024 + code, less 1032.
__device__ __forceinline__ uint32_t centred_low(uint32_t word) {
    const uint32_t a = mask_or(word, kLow, 0x64006400u), b = 0x64086408u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t centred_high(uint32_t word) {
    const uint32_t a = mask_or(word, kHigh, 0x64006400u), b = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// 16 H tokens, as H products: tk is the first one's place in the tile, pos its position.  MASKED: some row does not see
// all of them, or not all are there: those before position `seen`, where bit i of `pieces` is set for piece i of the tile
// (1 << piece_shift tokens).
template <int D, int NT, int H, bool MASKED>
__device__ __forceinline__ void att_step(AttRows<D, NT>& r, const uint8_t* K, const uint8_t* V, const uint32_t* KS, const uint32_t* VS, float key_scale,
                                         int tk, int pos, int seen, uint32_t pieces, int piece_shift) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // row m of a product is token m ^ (m / 2 % 2): the lanes that read values together then meet fewer banks twice
    const int pg = g ^ ((g >> 1) & 1);
    // the lane's scores: of product h, rows pg + 8 (i / 2), query rows 2 t + i % 2
    float x[H][NT][4] = {};
    uint32_t pk[H][2], pv[H][2];
    int at[H][2];
    uint32_t keys[H][2][D / 32];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int tok = tk + 16 * h + pg;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            pk[h][i] = KS[tok + 8 * i], pv[h][i] = VS[tok + 8 * i];
            if constexpr (MASKED) {
                at[h][i] = pos + 16 * h + pg + 8 * i;
                const bool ok = at[h][i] < seen && ((pieces >> ((tok + 8 * i) >> piece_shift)) & 1);
                if (!ok) pk[h][i] = pv[h][i] = 0, at[h][i] = 0x7FFFFFFF;   // what lies there is not looked at
            }
            load_words(keys[h][i], K + (tok + 8 * i) * (D / 2) + t * (D / 8));
        }
    }
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        uint4 q[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) q[nt] = r.q[(nt * (D / 32) + w) * 32];
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const uint32_t u = z ? keys[h][0][w] >> 8 : keys[h][0][w], v = z ? keys[h][1][w] >> 8 : keys[h][1][w];
                const uint32_t a0 = centred_low(u), a1 = centred_low(v), a2 = centred_high(u), a3 = centred_high(v);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(x[h][nt], a0, a1, a2, a3, z ? q[nt].z : q[nt].x, z ? q[nt].w : q[nt].y);
            }
    }
    // scores over a; `move`: one passes its row's reference by too much, or a value's step its bound
    float vstep[H][2], most = 0.0f;
    float2 steps[NT];   // the largest step, in magnitude, of a value that the row sees (MASKED), or that there is
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) steps[nt] = both(0.0f);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            vstep[h][i] = __uint_as_float(pv[h][i] << 16);
            if (!MASKED) steps[0].x = fmaxf(steps[0].x, fabsf(vstep[h][i]));
            const float s = __uint_as_float(pk[h][i] << 16);
            const float2 step = both(s * key_scale), middle = both(__fmaf_rn(8.0f, s, __uint_as_float(pk[h][i] & 0xFFFF0000u)) * key_scale);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float2 v = __ffma2_rn(make_float2(x[h][nt][2 * i], x[h][nt][2 * i + 1]), step, __fmul2_rn(middle, r.b[nt]));
                if (MASKED) {
                    if (at[h][i] == 0x7FFFFFFF || at[h][i] >= r.lim[nt][0]) v.x = -INFINITY;
                    if (at[h][i] == 0x7FFFFFFF || at[h][i] >= r.lim[nt][1]) v.y = -INFINITY;
                }
                x[h][nt][2 * i] = v.x, x[h][nt][2 * i + 1] = v.y;
                const float2 d = __ffma2_rn(v, r.a[nt], make_float2(-r.m[nt].x, -r.m[nt].y));
                if (!MASKED || v.x != -INFINITY) most = fmaxf(most, d.x);
                if (!MASKED || v.y != -INFINITY) most = fmaxf(most, d.y);
                if (MASKED && v.x != -INFINITY) steps[nt].x = fmaxf(steps[nt].x, fabsf(vstep[h][i]));
                if (MASKED && v.y != -INFINITY) steps[nt].y = fmaxf(steps[nt].y, fabsf(vstep[h][i]));
            }
        }
    bool wide = false;
#pragma unroll
    for (int nt = 0; nt < (MASKED ? NT : 1); ++nt) {
        const float2 c = MASKED ? r.c_of(nt) : both(r.c);
        wide |= steps[nt].x * c.x > 128.0f || (MASKED && steps[nt].y * c.y > 128.0f);
    }
    if (__any_sync(0xffffffffu, most > kAttSlack || wide)) {
        float2 c[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (MASKED || nt == 0) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {   // (a row's eight lanes)
                    steps[nt].x = fmaxf(steps[nt].x, __shfl_xor_sync(0xffffffffu, steps[nt].x, d));
                    if (MASKED) steps[nt].y = fmaxf(steps[nt].y, __shfl_xor_sync(0xffffffffu, steps[nt].y, d));
                }
            }
            if (!MASKED) steps[nt] = both(steps[0].x);
            // 128 over the power of two above the largest step
            const float2 old = MASKED ? r.c_of(nt) : both(r.c);
            c[nt] = old;
            if (steps[nt].x * old.x > 128.0f) c[nt].x = exp2_int(7 - min(static_cast<int>(__float_as_uint(steps[nt].x) >> 23) - 126, 127));
            if (steps[nt].y * old.y > 128.0f) c[nt].y = exp2_int(7 - min(static_cast<int>(__float_as_uint(steps[nt].y) >> 23) - 126, 127));
            const float2 scale_o = make_float2(power_ratio(c[nt].x, old.x), power_ratio(c[nt].y, old.y));
            float2 best = both(kAttNone);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (x[h][nt][2 * i] != -INFINITY) best.x = fmaxf(best.x, x[h][nt][2 * i] * r.a[nt].x);
                    if (x[h][nt][2 * i + 1] != -INFINITY) best.y = fmaxf(best.y, x[h][nt][2 * i + 1] * r.a[nt].y);
                }
#pragma unroll
            for (int d = 4; d < 32; d *= 2) {
                best.x = fmaxf(best.x, __shfl_xor_sync(0xffffffffu, best.x, d));
                best.y = fmaxf(best.y, __shfl_xor_sync(0xffffffffu, best.y, d));
            }
            const float2 m = make_float2(fmaxf(r.m[nt].x, best.x), fmaxf(r.m[nt].y, best.y));
            const float2 f = make_float2(ex2_approx(r.m[nt].x - m.x), ex2_approx(r.m[nt].y - m.y));
            r.m[nt] = m;
            r.l[nt] = __fmul2_rn(r.l[nt], f);
            r.lo[nt] = __fmul2_rn(r.lo[nt], f);
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) r.o[mt][nt][i] *= i & 1 ? f.y * scale_o.y : f.x * scale_o.x;
        }
        if constexpr (MASKED) {
            const float first = __shfl_sync(0xffffffffu, c[0].x, 0);
            bool same = true;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                same &= c[nt].x == first && c[nt].y == first;
                r.own_c()[nt * 32] = c[nt];   // (the lane's own)
            }
            r.apart = !__all_sync(0xffffffffu, same);
            r.c = first;
        } else {
            r.c = c[0].x;
        }
    }
    uint32_t pb[NT][2 * H];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 vs = both(vstep[h][i] * r.c), middle = both(__fmaf_rn(8.0f, vstep[h][i], __uint_as_float(pv[h][i] & 0xFFFF0000u)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 v = make_float2(x[h][nt][2 * i], x[h][nt][2 * i + 1]);
                const float2 d = __ffma2_rn(v, r.a[nt], make_float2(-r.m[nt].x, -r.m[nt].y));
                float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y)), w;
                if constexpr (MASKED) {   // step and least of a key that the row does not see may be NaN, and so may a
                    const bool x_in = v.x != -INFINITY, y_in = v.y != -INFINITY;
                    e = make_float2(x_in ? e.x : 0.0f, y_in ? e.y : 0.0f);
                    r.lo[nt] = make_float2(x_in ? __fmaf_rn(e.x, middle.x, r.lo[nt].x) : r.lo[nt].x, y_in ? __fmaf_rn(e.y, middle.y, r.lo[nt].y) : r.lo[nt].y);
                    w = make_float2(x_in ? e.x * (vstep[h][i] * r.c_of(nt).x) : 0.0f, y_in ? e.y * (vstep[h][i] * r.c_of(nt).y) : 0.0f);
                } else {
                    r.lo[nt] = __ffma2_rn(e, middle, r.lo[nt]);
                    w = __fmul2_rn(e, vs);
                }
                r.l[nt] = __fadd2_rn(r.l[nt], e);
                pb[nt][2 * h + i] = movmatrix(pair_of<__half>(w.x, w.y));
            }
        }
    // values: the lane's D / 8 dimensions (8 to a word) of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 in the products' order
    const int p0 = (2 * t) ^ (t & 1), p1 = (2 * t + 1) ^ (t & 1);
#pragma unroll
    for (int h = 0; h < H; ++h) {
        uint32_t v0[D / 64], v1[D / 64], v2[D / 64], v3[D / 64];
        const uint8_t* base = V + (tk + 16 * h) * (D / 2) + g * (D / 16);
        load_words(v0, base + p0 * (D / 2));
        load_words(v1, base + p1 * (D / 2));
        load_words(v2, base + (p0 + 8) * (D / 2));
        load_words(v3, base + (p1 + 8) * (D / 2));
#pragma unroll
        for (int w = 0; w < D / 64; ++w)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t u = __byte_perm(v0[w], v1[w], half ? 0x7632 : 0x5410), v = __byte_perm(v2[w], v3[w], half ? 0x7632 : 0x5410);
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const uint32_t us = z ? u >> 8 : u, vs = z ? v >> 8 : v;
                    const uint32_t a0 = centred_low(us), a1 = centred_high(us), a2 = centred_low(vs), a3 = centred_high(vs);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(r.o[4 * w + 2 * half + z][nt], a0, a1, a2, a3, pb[nt][2 * h], pb[nt][2 * h + 1]);
                }
            }
    }
}

// Where a unit lies.
struct AttItem {
    int b, head, n, rows, row0;
    int base, next;      // its first unit, and the one after its last
    int tiles;           // those that some row sees, one at least
    int seen;            // positions that some row sees
    int index;           // among all row tiles, with one new token per sequence
    long long token0, len;
};

template <int R>
__device__ __forceinline__ AttItem att_item(const AttParams& p, const int* first, int unit) {
    AttItem it;
    int lo = 0, hi = p.c.seqs;   // the last sequence whose units start at or before this one, and has some
    while (lo + 1 < hi) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= unit)
            lo = mid;
        else
            hi = mid;
    }
    it.b = lo;
    long long end;
    new_rows(p.c, lo, it.token0, end);
    it.n = static_cast<int>(end - it.token0);
    it.rows = it.n * p.per;
    it.len = p.c.lengths[lo];
    const long long cap = static_cast<long long>(p.c.width) << p.c.shift;
    const int seen = static_cast<int>(min(max(it.len, 0LL), cap));
    const int row_tiles = (it.rows + R - 1) / R;
    const int tiles = p.by_item ? 1 : kAttOver + max(1, (seen + kAttTile - 1) / kAttTile);
    const int rest = static_cast<int>(static_cast<unsigned>(unit - first[lo]) / static_cast<unsigned>(tiles));   // head and row tile
    it.head = row_tiles == 1 ? rest : rest / row_tiles;
    int tile = rest - it.head * row_tiles;
    it.base = first[lo] + rest * tiles;
    it.next = it.base + tiles;
    it.index = (lo * p.c.heads + it.head) * row_tiles + tile;
    if (p.by_item) tile = row_tiles - 1 - tile;   // the longest first
    it.row0 = tile * R;
    const int last = min(it.row0 + R, it.rows) - 1;
    it.seen = static_cast<int>(min(max(it.len - it.n + last / p.per + 1, 0LL), cap));
    it.tiles = max(1, (it.seen + kAttTile - 1) / kAttTile);
    return it;
}

// Tiles of an item among units beg .. end - 1.  An item's units are its overhead, then its tiles, then (of a tile of early rows)
// those that none of its rows sees.
__device__ __forceinline__ void att_tiles(const AttParams& p, const AttItem& it, int beg, int end, int& t0, int& t1) {
    if (p.by_item) {
        t0 = 0;
        t1 = it.tiles;
        return;
    }
    t0 = max(0, beg - it.base - kAttOver);
    t1 = min(it.tiles, end - it.base - kAttOver);
}

// The first unit of each sequence, and of all after the last one's, in shared memory; by all threads.
template <int R>
__device__ __forceinline__ void att_units(const AttParams& p, int* first, int threads) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long cap = static_cast<long long>(p.c.width) << p.c.shift;
    for (int b = threadIdx.x; b < p.c.seqs; b += threads) {
        long long beg, end;
        new_rows(p.c, b, beg, end);
        const int row_tiles = (static_cast<int>(end - beg) * p.per + R - 1) / R;
        const int seen = static_cast<int>(min(max(static_cast<long long>(p.c.lengths[b]), 0LL), cap));
        first[b + 1] = min(p.c.heads * row_tiles * (p.by_item ? 1 : kAttOver + max(1, (seen + kAttTile - 1) / kAttTile)), kAttUnits);
    }
    __syncthreads();
    if (warp == 0) {
        int sum = 0;
        for (int b0 = 0; b0 < p.c.seqs; b0 += 32) {
            int v = b0 + lane < p.c.seqs ? first[b0 + lane + 1] : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v = min(v + o, kAttUnits);
            }
            if (b0 + lane < p.c.seqs) first[b0 + lane + 1] = min(sum + v, kAttUnits);
            sum = min(sum + __shfl_sync(0xffffffffu, v, 31), kAttUnits);
        }
        if (lane == 0) first[0] = 0;
    }
    __syncthreads();
}

// This block's units: equal shares, the first `more` blocks one unit more; a unit each at least.
struct AttShare {
    int ctas, share, more, beg, end;
    __device__ __forceinline__ AttShare(const AttParams& p, int units) {
        const int cta = blockIdx.x;
        ctas = min(static_cast<int>(gridDim.x), units), share = ctas ? units / ctas : 0, more = units - share * ctas;
        beg = p.by_item ? min(cta, units) : cta < ctas ? cta * share + min(cta, more) : 0;
        end = p.by_item ? min(cta + 1, units) : cta < ctas ? beg + share + (cta < more) : 0;
    }
};

// What there is to join of a row tile that begins in this block: up to the owner of its last unit.
__device__ __forceinline__ AttDesc att_described(const AttItem& it, const AttShare& s, int cta, bool cut) {
    int last = -1;
    if (cut) {
        const int u1 = it.base + kAttOver + it.tiles - 1, big = s.more * (s.share + 1);
        last = min(u1 < big ? u1 / (s.share + 1) : s.more + (u1 - big) / s.share, s.ctas - 1);
    }
    return {cta, last, it.rows, it.head, it.row0, static_cast<int>(it.token0), {0, 0}};
}

template <int D, int NT, int RW>
__global__ void __launch_bounds__(kAttThreads, AttShape<D, NT, RW>::kPerSm) cache_attention_kernel(const AttParams p) {
    using Sh = AttShape<D, NT, RW>;
    constexpr int R = Sh::R, TW = Sh::TW, H = Sh::H;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::kStages + 2];
    __shared__ uint32_t there[Sh::kStages];
    __shared__ int dead;   // a wait ran out: nothing more is loaded
    float* join = reinterpret_cast<float*>(smem + Sh::kStages * Sh::kStage);
    uint8_t* queries = reinterpret_cast<uint8_t*>(join) + Sh::kJoin;
    float* stats = reinterpret_cast<float*>(queries + Sh::kQueries);
    int* first = reinterpret_cast<int*>(stats + Sh::kStats / 4);   // of each sequence, its first unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(bars), empty = full + 8 * Sh::kStages, q_full = empty + 8 * Sh::kStages, q_empty = q_full + 8, ring = smem_u32(smem);
    griddep_launch();
    if (threadIdx.x == 0) {
        for (int i = 0; i < Sh::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, kAttWarps);
        mbar_init(q_full, 1);
        mbar_init(q_empty, kAttWarps);
        fence_mbar_init();
        dead = 0;
    }
    griddep_wait();
    att_units<R>(p, first, kAttThreads);
    const int units = first[p.c.seqs], cta = blockIdx.x;
    const AttShare own(p, units);
    const int beg = own.beg, end = own.end;
    const int shift = min(p.c.shift, 7);   // tokens of a piece: a page, or a tile
    const int pieces = kAttTile >> shift;

    int stage = 0, phase = 0, item = 0;   // item: how many this block has had
    // Queries of all row tiles but the block's first, whose own loads begin as early.
    const auto ahead = [&](int i) { return Sh::kAhead && p.vec_q && i > 0; };
    if (warp == kAttWarps) {   // ---- the producer
        const long long half = D / 2;
        const uint32_t codes = static_cast<uint32_t>(half) << shift, pairs = 4u << shift;
        long long issued = 0;   // tiles
        for (int u = beg; u < end;) {
            const AttItem it = att_item<R>(p, first, u);
            int t0, t1;
            att_tiles(p, it, beg, end, t0, t1);
            u = it.next;
            if (t0 >= t1) continue;
            if (ahead(item)) {
                if (!mbar_wait_warp(q_empty, item & 1, p.wait_limit) && lane == 0) *p.err = ERR_WAIT_EMPTY, *static_cast<volatile int*>(&dead) = 1;
                if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&dead))) goto drain;
                const int rows = min(R, it.rows - it.row0);
                if (lane == 0) mbar_expect_tx(q_full, rows * D * 2);
                __syncwarp();
                for (int row = lane; row < rows; row += 32) {
                    const int i = (it.row0 + row) / p.per, j = it.row0 + row - i * p.per;
                    bulk_load(smem_u32(queries) + row * D * 2,
                              static_cast<const char*>(p.q) + 2 * ((it.token0 + i) * p.q_token + static_cast<long long>(it.head * p.per + j) * p.q_head), D * 2, q_full);
                }
            }
            ++item;
            const int per = 32 / pieces;   // tiles whose pages the lanes look up at once
            for (int tb = t0; tb < t1; tb += per) {
                const int mine = tb + lane / pieces;
                const long long pos = static_cast<long long>(mine) * kAttTile + (lane % pieces << shift);
                int page = -1;
                if (mine < t1 && pos < it.seen) page = page_of(p.c, it.b, pos);
                const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
                for (int i = 0; i < per && tb + i < t1; ++i) {
                    if (!mbar_wait_warp(empty + 8 * stage, phase ^ 1, p.wait_limit)) {
                        if (lane == 0) *p.err = ERR_WAIT_EMPTY, *static_cast<volatile int*>(&dead) = 1;
                    }
                    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&dead))) goto drain;
                    const uint32_t now = (have >> (i * pieces)) & ((1u << pieces) - 1);
                    if (lane == i * pieces) {
                        there[stage] = now;
                        const uint32_t bytes = __popc(now) * 2 * (codes + pairs);
                        if (bytes)
                            mbar_expect_tx(full + 8 * stage, bytes);
                        else
                            mbar_arrive(full + 8 * stage);
                    }
                    __syncwarp();
                    if (lane / pieces == i && page >= 0 && !(p.stall && it.base == 0 && mine == 0)) {   // (stall: the first tile of all)
                        const int at = lane % pieces << shift;                         // in the tile
                        const long long in = pos & (p.c.page - 1);                    // in the page
                        const uint32_t dst = ring + stage * Sh::kStage, bar = full + 8 * stage;
                        bulk_load(dst + at * (D / 2), p.c.k + page * p.c.k_page + it.head * p.c.k_head + in * half, codes, bar);
                        bulk_load(dst + Sh::kCodes + at * (D / 2), p.c.v + page * p.c.v_page + it.head * p.c.v_head + in * half, codes, bar);
                        bulk_load(dst + 2 * Sh::kCodes + at * 4, p.c.ks + page * p.c.ks_page + it.head * p.c.ks_head + in * 4, pairs, bar);
                        bulk_load(dst + 2 * Sh::kCodes + Sh::kPairs + at * 4, p.c.vs + page * p.c.vs_page + it.head * p.c.vs_head + in * 4, pairs, bar);
                    }
                    __syncwarp();
                    if (++stage == Sh::kStages) stage = 0, phase ^= 1;
                    ++issued;
                }
            }
        }
    drain:   // no copy is in flight when the block ends
        if (ahead(item - 1) && !mbar_wait_warp(q_full, item & 1, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
        for (long long i = max(0LL, issued - Sh::kStages); i < issued; ++i)
            if (!mbar_wait_warp(full + 8 * static_cast<int>(i % Sh::kStages), static_cast<int>(i / Sh::kStages) & 1, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
        return;
    }

    // ---- the computing warps
    const int rw = warp % RW, tw = warp / RW;   // which rows, which tokens of a tile
    const int g = lane >> 2, t = lane & 3;
    AttRows<D, NT> r;
    bool lost = false;
    if (!p.by_item && !p.listed && threadIdx.x == 0) p.desc[cta].last = -1;
    for (int u = beg; u < end;) {
        const AttItem it = att_item<R>(p, first, u);
        int t0, t1;
        att_tiles(p, it, beg, end, t0, t1);
        u = it.next;
        if (t0 >= t1) continue;
        const int row0 = it.row0 + rw * 8 * NT;
        const bool here = ahead(item);
        if (here && !lost && !mbar_wait_warp(q_full, (item & 1) ^ 1, p.wait_limit)) {
            lost = true;
            if (lane == 0) *p.err = ERR_WAIT_FULL, *static_cast<volatile int*>(&dead) = 1;
        }
        att_queries<D, NT>(p, r, reinterpret_cast<uint4*>(join + warp * (Sh::kWarp / 4)), it.token0, it.n, it.head, row0, it.rows, it.len,
                            here ? queries + rw * 8 * NT * D * 2 : nullptr);
        ++item;
        if (here) {
            __syncwarp();
            if (lane == 0) mbar_arrive(q_empty);
        }
        int all = it.seen;   // positions that all of the warp's rows see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) all = min(all, min(r.lim[nt][0], r.lim[nt][1]));
        all = __reduce_min_sync(0xffffffffu, all);
        for (int tile = t0; tile < t1; ++tile) {
            // (a warp that gives up goes on without loads, so that it meets the others at the segment's end)
            if (!lost && !mbar_wait_warp(full + 8 * stage, phase, p.wait_limit)) {
                lost = true;
                if (lane == 0) *p.err = ERR_WAIT_FULL, *static_cast<volatile int*>(&dead) = 1;
            }
            const uint8_t* K = smem + stage * Sh::kStage;
            const uint8_t* V = K + Sh::kCodes;
            const uint32_t* KS = reinterpret_cast<const uint32_t*>(V + Sh::kCodes);
            const uint32_t* VS = KS + kAttTile;
            const uint32_t have = there[stage];
            const bool whole = have == (1u << pieces) - 1;
            if (row0 < it.rows && !lost) {
#pragma unroll 1
                for (int tk = tw * 16 * H; tk < kAttTile; tk += TW * 16 * H) {
                    const int pos = tile * kAttTile + tk;
                    if (whole && pos + 16 * H <= all && !r.apart)
                        att_step<D, NT, H, false>(r, K, V, KS, VS, p.key_scale, tk, pos, it.seen, have, shift);
                    else if (pos < it.seen)
                        att_step<D, NT, H, true>(r, K, V, KS, VS, p.key_scale, tk, pos, it.seen, have, shift);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * stage);
            if (++stage == Sh::kStages) stage = 0, phase ^= 1;
        }
        // ---- the segment's end: the warps' numerators, references and sums meet in shared memory
        float2 c[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt] = r.c_of(nt);
        __syncwarp();   // all lanes are done with the queries, and what lies behind them
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float inv[2] = {power_ratio(1.0f, c[nt].x), power_ratio(1.0f, c[nt].y)};   // powers of two: exact
            float m[2] = {r.m[nt].x, r.m[nt].y}, l[2] = {r.l[nt].x, r.l[nt].y}, lo[2] = {r.lo[nt].x, r.lo[nt].y};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
                    lo[i] += __shfl_xor_sync(0xffffffffu, lo[i], d);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = (warp * NT + nt) * 8 + 2 * t + i;
                if (g == 0) stats[2 * row] = m[i], stats[2 * row + 1] = l[i];
                float* to = join + row * Sh::kPitch + g * (D / 8);
#pragma unroll
                for (int mt = 0; mt < D / 16; mt += 2)
                    *reinterpret_cast<float4*>(to + 2 * mt) =
                        make_float4(__fmaf_rn(r.o[mt][nt][i], inv[i], lo[i]), __fmaf_rn(r.o[mt][nt][2 + i] * 0.0625f, inv[i], lo[i]),
                                    __fmaf_rn(r.o[mt + 1][nt][i], inv[i], lo[i]), __fmaf_rn(r.o[mt + 1][nt][2 + i] * 0.0625f, inv[i], lo[i]));
            }
        }
        named_bar_sync(1, 32 * kAttWarps);
        const bool cut = t0 > 0 || t1 < it.tiles;
        const long long slot = 2LL * cta + (t0 == 0);   // an item begins in one CTA, and only one that began before ends in it
        const int rows = min(R, it.rows - it.row0);
        for (int i = threadIdx.x; i < rows * (D / 8); i += 32 * kAttWarps) {
            const int row = i / (D / 8), d = i % (D / 8) * 8;
            const int w0 = row / (8 * NT), in = row % (8 * NT);   // the warps that hold it: w0, w0 + RW, ..
            float m = kAttNone, l = 0.0f, y[8] = {};
#pragma unroll
            for (int z = 0; z < TW; ++z) m = fmaxf(m, stats[2 * ((w0 + z * RW) * 8 * NT + in)]);
#pragma unroll
            for (int z = 0; z < TW; ++z) {
                const int at = (w0 + z * RW) * 8 * NT + in;
                const float f = ex2_approx(stats[2 * at] - m);
                l = __fmaf_rn(f, stats[2 * at + 1], l);
                const float4 x0 = *reinterpret_cast<const float4*>(join + at * Sh::kPitch + d), x1 = *reinterpret_cast<const float4*>(join + at * Sh::kPitch + d + 4);
                y[0] = __fmaf_rn(f, x0.x, y[0]), y[1] = __fmaf_rn(f, x0.y, y[1]), y[2] = __fmaf_rn(f, x0.z, y[2]), y[3] = __fmaf_rn(f, x0.w, y[3]);
                y[4] = __fmaf_rn(f, x1.x, y[4]), y[5] = __fmaf_rn(f, x1.y, y[5]), y[6] = __fmaf_rn(f, x1.z, y[6]), y[7] = __fmaf_rn(f, x1.w, y[7]);
            }
            if (cut) {
                float* to = p.part + (slot * R + row) * D + d;
                reinterpret_cast<float4*>(to)[0] = make_float4(y[0], y[1], y[2], y[3]);
                reinterpret_cast<float4*>(to)[1] = make_float4(y[4], y[5], y[6], y[7]);
                if (d == 0) p.stat[2 * (slot * R + row)] = m, p.stat[2 * (slot * R + row) + 1] = l;
            } else {
                const int full_row = it.row0 + row, q = full_row / p.per;
                const long long at = (it.token0 + q) * p.o_token + static_cast<long long>(it.head * p.per + full_row - q * p.per) * p.o_head + d;
                const float div = l == 0.0f ? 0.0f : 1.0f / l;   // a row that sees nothing: zeros
#pragma unroll
                for (int z = 0; z < 8; ++z) y[z] *= div;
                if (p.type == Y_F16) {
                    __half* to = static_cast<__half*>(p.out) + at;
                    p.vec_o ? store8<__half, true>(to, y) : store8<__half, false>(to, y);
                } else {
                    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.out) + at;
                    p.vec_o ? store8<__nv_bfloat16, true>(to, y) : store8<__nv_bfloat16, false>(to, y);
                }
            }
        }
        named_bar_sync(1, 32 * kAttWarps);   // the buffer is free
        if (t0 == 0 && threadIdx.x == 0 && (p.listed || cut)) {   // the tile begins here: this CTA says what there is to join
            p.desc[p.listed ? it.index : cta] = att_described(it, own, cta, cut);
        }
    }
}

// Joins what a row tile's CTAs left: W warps a row, 32 parts of it at a time, each warp those that are its own modulo W.
constexpr int kAttJoinWide = 8;

template <int D, int W>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const AttParams p, int R) {
    constexpr int V = D / 32, ROWS = 8 / W;   // dimensions a lane, rows a block
    __shared__ float part[W > 1 ? W : 1][W > 1 ? D : 1], sums[W][2];
    // Only now: a next call's blocks that came while this kernel's still waited took SMs' room unevenly, and a few of its blocks
    // then ran after all others (32 sequences of up to 8192 tokens: 35 us a call instead of 27).
    griddep_wait();
    griddep_launch();
    const AttDesc a = p.desc[blockIdx.x];
    if (a.last < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = a.last - a.first + 1;
    for (int row = blockIdx.y * ROWS + warp / W; row < R && a.row0 + row < a.rows; row += gridDim.y * ROWS) {
        // part i: the first CTA's second, then the first one of each that follows
        const auto at = [&](int i) { return (2LL * (a.first + i) + (i == 0)) * R + row; };
        float m = kAttNone, l = 0.0f, y[V] = {};
        for (int i0 = warp % W; i0 < n; i0 += 32 * W) {
            const int mine = i0 + lane * W;
            const float2 stat = mine < n ? *reinterpret_cast<const float2*>(p.stat + 2 * at(mine)) : make_float2(kAttNone, 0.0f);
            float top = fmaxf(m, stat.x);
#pragma unroll
            for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float f = ex2_approx(m - top), w = mine < n ? ex2_approx(stat.x - top) : 0.0f;
            m = top;
            l = l * f + w * stat.y;   // the lane's share of the sum
#pragma unroll
            for (int z = 0; z < V; ++z) y[z] *= f;
            const int count = min(32, (n - i0 + W - 1) / W);
            constexpr int AT_ONCE = 4;
            for (int j0 = 0; j0 < count; j0 += AT_ONCE) {   // some parts' loads at once; those past the end are the last one's, with weight 0
                float v[AT_ONCE][V];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    const float* from = p.part + at(i0 + min(j0 + j, count - 1) * W) * D + lane;
#pragma unroll
                    for (int z = 0; z < V; ++z) v[j][z] = from[32 * z];
                }
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    const float wj = j0 + j < count ? __shfl_sync(0xffffffffu, w, j0 + j) : 0.0f;
#pragma unroll
                    for (int z = 0; z < V; ++z) y[z] = __fmaf_rn(wj, v[j][z], y[z]);
                }
            }
        }
#pragma unroll
        for (int d = 16; d; d /= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
        if constexpr (W > 1) {
            if (lane == 0) sums[warp][0] = m, sums[warp][1] = l;
#pragma unroll
            for (int z = 0; z < V; ++z) part[warp][z * 32 + lane] = y[z];
            __syncthreads();
            if (warp == 0) {
                float top = kAttNone;
#pragma unroll
                for (int w = 0; w < W; ++w) top = fmaxf(top, sums[w][0]);
                l = 0.0f;
#pragma unroll
                for (int z = 0; z < V; ++z) y[z] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float f = ex2_approx(sums[w][0] - top);
                    l = __fmaf_rn(f, sums[w][1], l);
#pragma unroll
                    for (int z = 0; z < V; ++z) y[z] = __fmaf_rn(f, part[w][z * 32 + lane], y[z]);
                }
            }
        }
        if (W == 1 || warp == 0) {
            const float div = l == 0.0f ? 0.0f : 1.0f / l;
            const int full_row = a.row0 + row, q = full_row / p.per;
            const long long to = static_cast<long long>(a.token0 + q) * p.o_token + static_cast<long long>(a.head * p.per + full_row - q * p.per) * p.o_head + lane;
#pragma unroll
            for (int z = 0; z < V; ++z) store_y(p.out, to + 32 * z, y[z] * div, p.type);
        }
        if constexpr (W > 1) __syncthreads();
    }
}

}  // namespace ptq8

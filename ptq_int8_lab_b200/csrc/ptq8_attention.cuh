// Attention over the cache of 4-bit keys and values.
//
// A code enters the tensor cores as it lies in the cache: four bits masked out of a word are, read as two f16, the
// subnormal numbers code * 2^-24 (or 16 code * 2^-24, the second code of a byte), exact, with no conversion at all.
// Five instructions widen eight codes; the powers of two, the steps and the least values go into the numbers around
// the products:
//   q . key    = step_k (q . codes) + least_k sum(q)                          queries as f16 times a power of two
//   sum p v    = sum (p step_v) codes + sum p least_v                         p step_v as f16, over a bound of step_v
// A query is scaled by the power of two that takes its largest value to 2^14 .. 2^15: f16 has three bits more than
// bf16, and what is more than 2^28 below the largest loses places only then.  p step_v is rounded to f16's 11 bits (an
// output has 11, or bf16's 8), with 2^-24 of the largest as its finest step; everything else is f32.
//
// A warp takes 16 tokens at a time as the rows of its products, 8 NT query rows (query token x head of a key's group) as
// the columns: keys codes [16 tokens x D] x queries [D x rows], then values codes [D x 16 tokens] x p [16 tokens x rows].
// Which of a lane's codes stands for which place of a product is free as long as both operands agree, so a lane reads
// its keys and values from the cache's own order, 4 D / 32 and 4 D / 64 words at a time.
//
// The softmax is kept running: a row's reference is moved only when a score passes it by 8 (in powers of two), a vote of
// the warp that fails almost always, and the sums of 8 lanes meet at the end of a segment.
//
// Work is units of 64 tokens of one key head and row tile.  All sequences' units lie in one order, and CTA c of N takes
// those from c U / N to (c + 1) U / N: equal shares whatever the lengths are, known on the device only.  A row tile cut
// by a share's end leaves (numerators, reference, sum) in the workspace, and a second kernel joins them.
// A producer warp keeps bulk copies of whole tiles in flight; four warps compute, RW of them on different rows, 4 / RW on
// different tokens of a tile.
#pragma once

#include "ptq8_cache.cuh"
#include "ptq8_linear.cuh"

namespace ptq8 {

constexpr int kAttTile = 64, kAttWarps = 4, kAttThreads = 32 * (kAttWarps + 1);
constexpr float kAttNone = -1e30f;   // reference of a row that has seen nothing
constexpr float kAttSlack = 8.0f;

struct AttDesc {
    int slot, last;        // first partial result of the row tile, the last CTA that has one (-1: nothing to join)
    int rows, head;        // of this tile; the key head
    long long token0;      // of its sequence
    int row0, pad;
};

struct AttParams {
    CacheView c;
    const void* q;
    void* out;
    long long q_token, q_head, o_token, o_head;   // elements
    float scale_log2;   // scale * log2(e)
    int per;            // query heads of a key head
    int by_item;        // 1: a CTA per row tile, none cut; 0: equal shares
    int type;           // Y_F16 or Y_BF16
    int vec_q, vec_o;   // rows at multiples of 16 bytes
    float* part;        // [2 N][R][D] numerators
    float* stat;        // [2 N][R][2] reference, sum
    AttDesc* desc;      // [N]
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

template <int D, int NT, int RW>
struct AttShape {
    static constexpr int R = 8 * NT * RW, TW = kAttWarps / RW;
    static constexpr int kPerSm = D * NT <= 128 ? 3 : 2;
    static constexpr int kStages = 4;
    static constexpr int kCodes = kAttTile * D / 2, kPairs = kAttTile * 4, kStage = 2 * (kCodes + kPairs);
    static constexpr int kPitch = D + 4;   // floats of a row of the joining buffer, off the banks' period
    static constexpr int kJoin = kAttWarps * 8 * NT * kPitch * 4, kStats = kAttWarps * 8 * NT * 2 * 4;
    static constexpr int smem(int seqs) { return kStages * kStage + kJoin + kStats + (seqs + 1) * 8 + 128; }
};

// A warp's query rows and what it has of their softmax.  Lane (g, t) = (lane / 4, lane % 4) holds, for the products,
// row g of each tile of 8; of the sums, rows 2 t and 2 t + 1.
template <int D, int NT>
struct AttRows {
    uint32_t q[NT][D / 32][4];
    float a[NT][2], b[NT][2];            // score in powers of two = a * (step (q . codes) + least b)
    float m[NT][2], l[NT][2], lo[NT][2]; // reference, sum of p, sum of p least_v
    int lim[NT][2];                      // positions that the row sees
    float o[D / 16][NT][4];
    float c;                             // what p step_v is multiplied by: a power of two
};

__device__ __forceinline__ float att_value(const void* p, long long at, int type) {
    return type == Y_F16 ? __half2float(static_cast<const __half*>(p)[at]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

// The lane's part of the query rows from `row` on: D / 4 values of each tile's row g.
template <int D, int NT>
__device__ __forceinline__ void att_queries(const AttParams& p, AttRows<D, NT>& r, long long token0, int n, int head, int row0, int rows, long long len) {
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
#pragma unroll
                for (int k = 0; k < DL / 8; ++k) {
                    float e[8];
                    if (p.type == Y_F16)
                        load8<__half, true>(static_cast<const __half*>(p.q) + at + 8 * k, e);
                    else
                        load8<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(p.q) + at + 8 * k, e);
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
        // 2^e takes the largest to 2^14 .. 2^15 (rows below 2^-86 stay below; their scores are zero for any key)
        const int e = min(max(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100);
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
            r.q[nt][w][0] = pair_of<__half>(x[0], x[4]);
            r.q[nt][w][1] = pair_of<__half>(x[1] * 0.0625f, x[5] * 0.0625f);
            r.q[nt][w][2] = pair_of<__half>(x[2], x[6]);
            r.q[nt][w][3] = pair_of<__half>(x[3] * 0.0625f, x[7] * 0.0625f);
        }
        // the products are 2^(e - 24) of the true ones; NaN and infinities in a row make all of its scores NaN
        const float a = isfinite(top) ? exp2_int(24 - e) * p.scale_log2 : __int_as_float(0x7FC00000);
        const float b = sum * 0x1p-24f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int src = (2 * t + i) * 4, my = row0 + nt * 8 + 2 * t + i;
            r.a[nt][i] = __shfl_sync(0xffffffffu, a, src);
            r.b[nt][i] = __shfl_sync(0xffffffffu, b, src);
            r.m[nt][i] = kAttNone;
            r.l[nt][i] = r.lo[nt][i] = 0.0f;
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
}

constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;

// 16 tokens: tk is the first one's place in the tile, pos its position.  MASKED: some row does not see all of them, or
// not all are there: `there` tokens from tk on, and where bit i of `pieces` is not set those of piece i (1 << shift tokens).
template <int D, int NT, bool MASKED>
__device__ __forceinline__ void att_step(AttRows<D, NT>& r, const uint8_t* K, const uint8_t* V, const uint32_t* KS, const uint32_t* VS, int tk,
                                         int pos, int seen, uint32_t pieces, int piece_shift) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // row m of a product is token m ^ (m / 2 % 2): the lanes that read values together then meet fewer banks twice
    const int pg = g ^ ((g >> 1) & 1);
    uint32_t ka[D / 32], kb[D / 32];
    load_words(ka, K + (tk + pg) * (D / 2) + t * (D / 8));
    load_words(kb, K + (tk + pg + 8) * (D / 2) + t * (D / 8));
    uint32_t pk[2] = {KS[tk + pg], KS[tk + pg + 8]}, pv[2] = {VS[tk + pg], VS[tk + pg + 8]};
    int at[2];
    if constexpr (MASKED) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            at[i] = pos + pg + 8 * i;
            const bool ok = at[i] < seen && ((pieces >> ((tk + pg + 8 * i) >> piece_shift)) & 1);
            if (!ok) pk[i] = pv[i] = 0, at[i] = 0x7FFFFFFF;   // what lies there is not looked at
        }
    }
    float s[NT][4] = {}, s2[NT][4] = {};
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], ka[w] & kLow, kb[w] & kLow, ka[w] & kHigh, kb[w] & kHigh, r.q[nt][w][0], r.q[nt][w][1]);
        const uint32_t x = ka[w] >> 8, y = kb[w] >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816(s2[nt], x & kLow, y & kLow, x & kHigh, y & kHigh, r.q[nt][w][2], r.q[nt][w][3]);
    }
    float vstep[2], vleast[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) vstep[i] = __uint_as_float(pv[i] << 16), vleast[i] = __uint_as_float(pv[i] & 0xFFFF0000u);
    // scores over a, then their distance to the reference in powers of two
    bool move = fmaxf(vstep[0], vstep[1]) * r.c > 128.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tok = i >> 1, row = i & 1;
            const float step = __uint_as_float(pk[tok] << 16), least = __uint_as_float(pk[tok] & 0xFFFF0000u);
            float x = __fmaf_rn(s[nt][i] + s2[nt][i], step, least * r.b[nt][row]);
            if (MASKED && (at[tok] == 0x7FFFFFFF || at[tok] >= r.lim[nt][row])) x = -INFINITY;
            s[nt][i] = x;
            s2[nt][i] = __fmaf_rn(x, r.a[nt][row], -r.m[nt][row]);
            if (MASKED && x == -INFINITY) s2[nt][i] = -INFINITY;   // (a is NaN for a row that is not finite)
            move = move || s2[nt][i] > kAttSlack;
        }
    if (__any_sync(0xffffffffu, move)) {
        float top = fmaxf(vstep[0], vstep[1]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // all lanes of the warp hold the same bound: 128 over the power of two above it
        float scale_o = 1.0f;
        if (top * r.c > 128.0f) {
            const int e = min(static_cast<int>(__float_as_uint(top) >> 23) - 126, 127);
            const float c = exp2_int(7 - e);
            scale_o = c / r.c;
            r.c = c;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int row = 0; row < 2; ++row) {
                // (scores anew: beside the first reference their distance to it has no places left)
                float best = kAttNone;
                if (s[nt][row] != -INFINITY) best = fmaxf(best, s[nt][row] * r.a[nt][row]);
                if (s[nt][2 + row] != -INFINITY) best = fmaxf(best, s[nt][2 + row] * r.a[nt][row]);
#pragma unroll
                for (int d = 4; d < 32; d *= 2) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
                const float m = fmaxf(r.m[nt][row], best);
                f[row] = ex2_approx(r.m[nt][row] - m);
                r.m[nt][row] = m;
                r.l[nt][row] *= f[row];
                r.lo[nt][row] *= f[row];
                s2[nt][row] = s[nt][row] == -INFINITY ? -INFINITY : __fmaf_rn(s[nt][row], r.a[nt][row], -m);
                s2[nt][2 + row] = s[nt][2 + row] == -INFINITY ? -INFINITY : __fmaf_rn(s[nt][2 + row], r.a[nt][row], -m);
            }
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) r.o[mt][nt][i] *= f[i & 1] * scale_o;
        }
    }
    uint32_t pb[NT][2];
    const float vs[2] = {vstep[0] * r.c, vstep[1] * r.c};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = ex2_approx(s2[nt][i]);
            const int tok = i >> 1, row = i & 1;
            if (MASKED && s2[nt][i] == -INFINITY) {   // step and least of a key that the row does not see may be NaN
                w[i] = 0.0f;
            } else {
                r.l[nt][row] += e;
                r.lo[nt][row] = __fmaf_rn(e, vleast[tok], r.lo[nt][row]);
                w[i] = e * vs[tok];
            }
        }
        pb[nt][0] = movmatrix(pair_of<__half>(w[0], w[1]));
        pb[nt][1] = movmatrix(pair_of<__half>(w[2], w[3]));
    }
    // values: the lane's D / 8 dimensions (8 to a word) of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 in the products' order
    const int p0 = (2 * t) ^ (t & 1), p1 = (2 * t + 1) ^ (t & 1);
    uint32_t v0[D / 64], v1[D / 64], v2[D / 64], v3[D / 64];
    const uint8_t* base = V + tk * (D / 2) + g * (D / 16);
    load_words(v0, base + p0 * (D / 2));
    load_words(v1, base + p1 * (D / 2));
    load_words(v2, base + (p0 + 8) * (D / 2));
    load_words(v3, base + (p1 + 8) * (D / 2));
#pragma unroll
    for (int w = 0; w < D / 64; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(v0[w], v1[w], half ? 0x7632 : 0x5410), y = __byte_perm(v2[w], v3[w], half ? 0x7632 : 0x5410);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const uint32_t xs = z ? x >> 8 : x, ys = z ? y >> 8 : y;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(r.o[4 * w + 2 * half + z][nt], xs & kLow, xs & kHigh, ys & kLow, ys & kHigh, pb[nt][0], pb[nt][1]);
            }
        }
}

// Where a unit lies.
struct AttItem {
    int b, head;
    long long token0, len, base;   // base: its first unit
    int n, rows, row0, tiles;      // tiles: those that some row sees, one at least
    int seen;                      // positions that some row sees
};

template <int R>
__device__ __forceinline__ AttItem att_item(const AttParams& p, const long long* first, long long unit) {
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
    const long long tiles = p.by_item ? 1 : max(1, (seen + kAttTile - 1) / kAttTile);
    const long long rest = unit - first[lo];
    it.head = static_cast<int>(rest / (row_tiles * tiles));
    int tile = static_cast<int>((rest - it.head * (row_tiles * tiles)) / tiles);
    it.base = first[lo] + (it.head * static_cast<long long>(row_tiles) + tile) * tiles;
    if (p.by_item) tile = row_tiles - 1 - tile;   // the longest first
    it.row0 = tile * R;
    const int last = min(it.row0 + R, it.rows) - 1;
    it.seen = static_cast<int>(min(max(it.len - it.n + last / p.per + 1, 0LL), cap));
    it.tiles = max(1, (it.seen + kAttTile - 1) / kAttTile);
    return it;
}

template <int D, int NT, int RW>
__global__ void __launch_bounds__(kAttThreads, AttShape<D, NT, RW>::kPerSm) cache_attention_kernel(const AttParams p) {
    using Sh = AttShape<D, NT, RW>;
    constexpr int R = Sh::R, TW = Sh::TW;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::kStages];
    __shared__ uint32_t there[Sh::kStages];
    __shared__ int dead;   // a wait ran out: nothing more is loaded
    float* join = reinterpret_cast<float*>(smem + Sh::kStages * Sh::kStage);
    float* stats = join + Sh::kJoin / 4;
    long long* first = reinterpret_cast<long long*>(stats + Sh::kStats / 4);   // of each sequence, its first unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(bars), empty = full + 8 * Sh::kStages, ring = smem_u32(smem);
    griddep_launch();
    if (threadIdx.x == 0) {
        for (int i = 0; i < Sh::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, kAttWarps);
        fence_mbar_init();
        dead = 0;
    }
    griddep_wait();
    const long long cap = static_cast<long long>(p.c.width) << p.c.shift;
    for (int b = threadIdx.x; b < p.c.seqs; b += kAttThreads) {
        long long beg, end;
        new_rows(p.c, b, beg, end);
        const long long row_tiles = ((end - beg) * p.per + R - 1) / R;
        const long long seen = min(max(static_cast<long long>(p.c.lengths[b]), 0LL), cap);
        first[b + 1] = p.c.heads * row_tiles * (p.by_item ? 1 : max(1LL, (seen + kAttTile - 1) / kAttTile));
    }
    __syncthreads();
    if (warp == 0) {
        long long sum = 0;
        for (int b0 = 0; b0 < p.c.seqs; b0 += 32) {
            long long v = b0 + lane < p.c.seqs ? first[b0 + lane + 1] : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const long long o = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += o;
            }
            if (b0 + lane < p.c.seqs) first[b0 + lane + 1] = sum + v;
            sum += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) first[0] = 0;
    }
    __syncthreads();
    const long long units = first[p.c.seqs], cta = blockIdx.x, ctas = min(static_cast<long long>(gridDim.x), units);   // a unit each at least
    const long long beg = p.by_item ? min(cta, units) : cta < ctas ? cta * units / ctas : 0, end = p.by_item ? min(cta + 1, units) : cta < ctas ? (cta + 1) * units / ctas : 0;
    const int shift = min(p.c.shift, 6);   // tokens of a piece: a page, or a tile
    const int pieces = kAttTile >> shift;

    int stage = 0, phase = 0;
    if (warp == kAttWarps) {   // ---- the producer
        const long long half = D / 2;
        const uint32_t codes = static_cast<uint32_t>(half) << shift, pairs = 4u << shift;
        long long issued = 0;   // tiles
        for (long long u = beg; u < end;) {
            const AttItem it = att_item<R>(p, first, u);
            const int t0 = static_cast<int>(u - it.base);
            const long long left = it.base + (p.by_item ? 1 : max(1LL, (min(max(it.len, 0LL), cap) + kAttTile - 1) / kAttTile));   // the item's last unit + 1
            const int t1 = p.by_item ? it.tiles : static_cast<int>(min(static_cast<long long>(it.tiles), end - it.base));
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
                    if (lane / pieces == i && page >= 0 && !(p.stall && cta == 0 && u == beg && tb == t0 && i == 0)) {
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
            u = left;
        }
    drain:   // no copy is in flight when the block ends
        for (long long i = max(0LL, issued - Sh::kStages); i < issued; ++i)
            if (!mbar_wait_warp(full + 8 * static_cast<int>(i % Sh::kStages), static_cast<int>(i / Sh::kStages) & 1, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
        return;
    }

    // ---- the computing warps
    const int rw = warp % RW, tw = warp / RW;   // which rows, which tokens of a tile
    const int g = lane >> 2, t = lane & 3;
    AttRows<D, NT> r;
    bool lost = false;
    if (!p.by_item && threadIdx.x == 0) p.desc[cta].last = -1;
    for (long long u = beg; u < end;) {
        const AttItem it = att_item<R>(p, first, u);
        const int t0 = static_cast<int>(u - it.base);
        const long long left = it.base + (p.by_item ? 1 : max(1LL, (min(max(it.len, 0LL), cap) + kAttTile - 1) / kAttTile));
        const int t1 = p.by_item ? it.tiles : static_cast<int>(min(static_cast<long long>(it.tiles), end - it.base));
        u = left;
        if (t0 >= t1) continue;   // units that no row of the tile sees
        const int row0 = it.row0 + rw * 8 * NT;
        att_queries<D, NT>(p, r, it.token0, it.n, it.head, row0, it.rows, it.len);
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
                for (int tk = tw * 16; tk < kAttTile; tk += TW * 16) {
                    const int pos = tile * kAttTile + tk;
                    if (whole && pos + 16 <= all)
                        att_step<D, NT, false>(r, K, V, KS, VS, tk, pos, it.seen, have, shift);
                    else if (pos < it.seen)
                        att_step<D, NT, true>(r, K, V, KS, VS, tk, pos, it.seen, have, shift);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * stage);
            if (++stage == Sh::kStages) stage = 0, phase ^= 1;
        }
        // ---- the segment's end: the warps' numerators, references and sums meet in shared memory
        named_bar_sync(1, 32 * kAttWarps);   // the buffer is free
        const float inv = 1.0f / r.c;        // a power of two: exact
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {
                    r.l[nt][i] += __shfl_xor_sync(0xffffffffu, r.l[nt][i], d);
                    r.lo[nt][i] += __shfl_xor_sync(0xffffffffu, r.lo[nt][i], d);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = (warp * NT + nt) * 8 + 2 * t + i;
                if (g == 0) stats[2 * row] = r.m[nt][i], stats[2 * row + 1] = r.l[nt][i];
                float* to = join + row * Sh::kPitch + g * (D / 8);
#pragma unroll
                for (int mt = 0; mt < D / 16; mt += 2)
                    *reinterpret_cast<float4*>(to + 2 * mt) =
                        make_float4(__fmaf_rn(r.o[mt][nt][i] * 0x1p24f, inv, r.lo[nt][i]), __fmaf_rn(r.o[mt][nt][2 + i] * 0x1p20f, inv, r.lo[nt][i]),
                                    __fmaf_rn(r.o[mt + 1][nt][i] * 0x1p24f, inv, r.lo[nt][i]), __fmaf_rn(r.o[mt + 1][nt][2 + i] * 0x1p20f, inv, r.lo[nt][i]));
            }
        }
        named_bar_sync(1, 32 * kAttWarps);
        const bool cut = t0 > 0 || t1 < it.tiles;
        const long long slot = 2 * cta + (it.base < beg || t0 > 0 ? 0 : it.base > beg ? 1 : 0);
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
        if (cut && t0 == 0 && threadIdx.x == 0) {   // the tile begins here: this CTA says what there is to join
            const long long last = it.base + it.tiles - 1;   // its owner: the c with c U / N <= last < (c + 1) U / N
            p.desc[cta] = {static_cast<int>(slot), static_cast<int>(((last + 1) * ctas - 1) / units), it.rows, it.head, it.token0, it.row0, 0};
        }
    }
}

// Joins what a row tile's CTAs left.  A block a row, eight warps on different parts of it.
template <int D>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const AttParams p, int R) {
    constexpr int V = D / 32;   // dimensions a lane
    __shared__ float part[8][D], sums[8][2];
    griddep_launch();
    griddep_wait();
    const AttDesc a = p.desc[blockIdx.x];
    const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.last < 0 || a.row0 + row >= a.rows) return;
    const int n = a.last - static_cast<int>(blockIdx.x) + 1;
    // part i: this CTA's, then the first one of each that follows
    const auto slot = [&](int i) { return static_cast<long long>(i == 0 ? a.slot : 2 * (static_cast<int>(blockIdx.x) + i)); };
    float m = kAttNone, l = 0.0f, y[V] = {};
    for (int i = warp; i < n; i += 8) {
        const long long at = slot(i) * R + row;
        const float mi = p.stat[2 * at], li = p.stat[2 * at + 1];
        const float up = fmaxf(m, mi), f = ex2_approx(m - up), fi = ex2_approx(mi - up);
        m = up;
        l = l * f + li * fi;
#pragma unroll
        for (int z = 0; z < V; ++z) y[z] = y[z] * f + fi * p.part[at * D + z * 32 + lane];
    }
#pragma unroll
    for (int z = 0; z < V; ++z) part[warp][z * 32 + lane] = y[z];
    if (lane == 0) sums[warp][0] = m, sums[warp][1] = l;
    __syncthreads();
    if (threadIdx.x >= D) return;
    float top = kAttNone;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, sums[w][0]);
    float s = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const float f = ex2_approx(sums[w][0] - top);
        s = __fmaf_rn(f, sums[w][1], s);
        v = __fmaf_rn(f, part[w][threadIdx.x], v);
    }
    v = s == 0.0f ? 0.0f : v / s;
    const int full_row = a.row0 + row, q = full_row / p.per;
    store_y(p.out, (a.token0 + q) * p.o_token + static_cast<long long>(a.head * p.per + full_row - q * p.per) * p.o_head + threadIdx.x, v, p.type);
}

}  // namespace ptq8

// Attention over the cache of 4-bit keys and values for many query rows: tcgen05.
//
// The mathematics are those of the kernel for few rows (codes as f16, steps and least values around the products); here
//   S = Q' (codes_k - 8)^T     128 rows x 128 tokens, Q' in shared memory, f32 in TMEM
//   O += P (codes_v - 8)       P = p step_v c as f16 in TMEM where S was, O in TMEM
// with code - 8 as normal f16 numbers (16 (code - 8) for the second code of a byte, whose queries are a sixteenth).  The codes are
// widened to f16 once for 256 rows: a cached tile of 128 tokens becomes two operands of 32 KB (D = 128), keys and values in
// the same order, a token's row of 64 dimensions to 128 bytes: read as K-major for S, as N-major for O.  Where a word's
// eight codes stand for dimensions in another order (0 4 1 5 2 6 3 7), queries and outputs follow it.
//
// A thread owns a row: no value of a softmax leaves it.  It goes over its 128 scores once, 16 at a time, with the reference that it
// has; only where one passes that by 2^8 (or a value's step its bound) does it go over P so far and O with a new one, a
// whole power of two away, so that P changes exactly.
//
// Warps: 0-3 and 4-7 softmax of 128 rows each, in turns with the tensor core: one's products run while the other's
// exponentials do; 8-11 widen codes; 12 issues MMAs; 13 copies tiles in; 14, 15 idle.
//
// What bounds it: the softmax's instructions.  2 x 512 new tokens of 32 heads (8 key heads, D = 128, bf16) over 4500 to 8192
// positions take 247 us, 413 TFLOP/s, against 463 us with warp-level products; a tile of 128 tokens takes some 7700 cycles, of
// which the tensor cores need 2000 and the exponentials 2000 (4 a cycle and scheduler); the rest are the other twelve instructions for
// two scores and what they wait for, with two warps of the softmax a scheduler.  All eight steps of a tile's loop written out, 32 KB of
// instructions, waited for those (285 us where this took 243).  The kernel spills 68 bytes (132 of loads).  The tokens' pairs as they lie in the cache, half the bytes from shared memory for four more instructions
// for two scores: 270.  More registers for the softmax warps by setmaxnreg: 559, the others spilled.
#pragma once

#include "ptq8_attention.cuh"

namespace ptq8 {

constexpr int kTcRows = 256, kTcThreads = 512;

template <int D>
struct TcAttShape {
    static constexpr int kStages = 3;
    static constexpr int kCodes = kAttTile * D / 2, kPairs = kAttTile * 4, kStage = 2 * (kCodes + kPairs);
    static constexpr int kBlock = kAttTile * 128;              // 64 dimensions of 128 rows or tokens as f16
    static constexpr int kHalf = D / 64 * kBlock;              // an operand
    static constexpr int kParam = kAttTile * 16 + 32;          // of a tile: by 16 tokens, for each two step_k, middle_k, and for each two step_v, middle_v; then which there are, and the warps' largest steps
    static constexpr int smem(int seqs) { return 1024 + 5 * kHalf + kStages * kStage + 2 * kParam + (seqs + 1) * 4; }
    static_assert(smem(1024) + 1024 <= 227 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_load8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}
// (naming the registers: their uses stay behind it)
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])::"memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A B^T, f16 -> f32; A in shared memory or in TMEM.  By one lane of a converged warp.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// f32 accumulators of f16 operands, A K-major, B K-major or N-major, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool n_major) {
    return (1u << 4) | (n_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}
// N-major operand: 8 tokens of 64 dimensions in 1024 bytes, the next 64 dimensions a block further.
__device__ __forceinline__ uint64_t n_major_desc(uint32_t saddr, uint32_t block) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | static_cast<uint64_t>(block >> 4) << 16 | static_cast<uint64_t>(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// A thread's row of the softmax.
struct TcRow {
    float a, b, m, l, lo, c;   // as in AttRows
    int lim;
    bool fresh;                // it has seen nothing: m is 0, and says nothing
};

// New references, whole powers of two from the old ones (`up` of them; P so far changes exactly), and new c: what there is of P (the
// first `cols` columns at s) and O (`ocols` columns at o) follows.  By a whole warp.
__device__ __noinline__ void tc_rescale(uint32_t s, int cols, uint32_t o, int ocols, float scale) {
    __syncwarp();
    tmem_stored();
#pragma unroll 1
    for (int i = 0; i < cols; i += 8) {
        uint32_t x[8];
        tmem_load8(s + i, x);
        tmem_wait_ld(x);
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x[z]));   // (a scale below 2^-24 is no f16 number, its product may be)
            x[z] = pair_of<__half>(v.x * scale, v.y * scale);
        }
        tmem_store8(s + i, x);
    }
#pragma unroll 1
    for (int i = 0; i < ocols; i += 8) {
        uint32_t x[8];
        tmem_load8(o + i, x);
        tmem_wait_ld(x);
#pragma unroll
        for (int z = 0; z < 8; ++z) x[z] = __float_as_uint(__uint_as_float(x[z]) * scale);
        tmem_store8(o + i, x);
    }
    tmem_stored();
}

// Of 16 tokens of a tile, the k-th ones: their scores over a, the most of them and the largest step; `in` says which the row sees (MASKED).
template <bool MASKED>
__device__ __forceinline__ void tc_scores(const TcRow& r, const uint32_t (&x)[16], const float4* param, int k, uint32_t in, float2 (&v)[8], float& most, float& steps) {
    const float2 b = both(r.b);
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 key = param[16 * k + i];
        v[i] = __ffma2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), make_float2(key.x, key.y), __fmul2_rn(make_float2(key.z, key.w), b));
        if constexpr (MASKED) {   // (what a row does not see may be NaN)
            if (!((in >> (2 * i)) & 1)) v[i].x = -INFINITY;
            if (!((in >> (2 * i + 1)) & 1)) v[i].y = -INFINITY;
            const float4 value = param[16 * k + 8 + i];
            if ((in >> (2 * i)) & 1) steps = fmaxf(steps, fabsf(value.x));
            if ((in >> (2 * i + 1)) & 1) steps = fmaxf(steps, fabsf(value.y));
        }
        most = fmaxf(most, fmaxf(v[i].x, v[i].y));
    }
}

// The row's 128 scores of a tile at s become P there.  MASKED: some row does not see all of the tile's tokens.  largest: the tile's largest step.
template <bool MASKED>
__device__ __forceinline__ void tc_tile(TcRow& r, uint32_t s, uint32_t o, int ocols, const float4* param, const uint32_t* there, int pos, float largest) {
    float2 sum = make_float2(r.l, 0.0f), low = make_float2(r.lo, 0.0f);
    const auto seen = [&](int k) {
        if (!MASKED) return 0xFFFFu;
        const int n = min(max(r.lim - pos - 16 * k, 0), 16);
        return (there[k >> 1] >> (16 * (k & 1))) & ((1u << n) - 1);
    };
    // A new reference where one is wanted, before the k-th 16 scores become P.  (Scores are kept as they are until then: a difference from a
    // reference far below them would say only roughly how far they are from the new one.)
    const auto check = [&](int k, float2 (&v)[8], float most, float steps, uint32_t (&coming)[16]) {
        const float top = most * r.a;   // (a: a power of two)
        const bool move = top - r.m > kAttSlack || (r.fresh && top > kAttNone);
        if (__any_sync(0xffffffffu, move || steps * r.c > 128.0f)) {
            tmem_wait_ld(coming);   // registers that a load has yet to write do not go through a call
            float f = 1.0f;
            if (move) {
                const float m = ceilf(top);
                if (!r.fresh) f = exp2_int(static_cast<int>(fmaxf(r.m - m, -126.0f)));
                r.m = m, r.fresh = false;
            }
            float c = r.c;
            if (steps * r.c > 128.0f) c = exp2_int(7 - min(static_cast<int>(__float_as_uint(steps) >> 23) - 126, 127));
            tc_rescale(s, 8 * k, o, ocols, f * power_ratio(c, r.c));
            r.c = c;
            sum = __fmul2_rn(sum, both(f)), low = __fmul2_rn(low, both(f));
        }
        const uint32_t in = seen(k);
        const float2 a = both(r.a), m = both(-r.m);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = __ffma2_rn(v[i], a, m);
            if constexpr (MASKED) {   // (a may be zero or NaN)
                if (!((in >> (2 * i)) & 1)) v[i].x = -INFINITY;
                if (!((in >> (2 * i + 1)) & 1)) v[i].y = -INFINITY;
            }
        }
    };
    // 16 scores at a time: while some become P, the next ones are looked at and the ones after those are on their way
    uint32_t x[2][16];
    float2 v[2][8];
    float most, steps = MASKED ? 0.0f : largest;
    tmem_ld16(s, x[0]);
    tmem_wait_ld(x[0]);
    tmem_ld16(s + 16, x[1]);
    tc_scores<MASKED>(r, x[0], param, 0, seen(0), v[0], most, steps);
    check(0, v[0], most, steps, x[1]);
#pragma unroll 2   // (all eight in a row, 32 KB of instructions that a warp goes through once a tile, wait for them)
    for (int k = 0; k < 8; ++k) {
        steps = 0.0f;
        if (k < 7) {
            tmem_wait_ld(x[(k + 1) & 1]);
            if (k < 6) tmem_ld16(s + 16 * (k + 2), x[k & 1]);
            tc_scores<MASKED>(r, x[(k + 1) & 1], param, k + 1, seen(k + 1), v[(k + 1) & 1], most, steps);
        }
        const uint32_t in = seen(k);
        const float2 c = both(r.c);
        uint32_t P[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float4 value = param[16 * k + 8 + i];
            if constexpr (MASKED) {
                if (!((in >> (2 * i)) & 1)) value.x = value.z = 0.0f;
                if (!((in >> (2 * i + 1)) & 1)) value.y = value.w = 0.0f;
            }
            const float2 e = make_float2(ex2_approx(v[k & 1][i].x), ex2_approx(v[k & 1][i].y));
            sum = __fadd2_rn(sum, e);
            low = __ffma2_rn(e, make_float2(value.z, value.w), low);
            const float2 w = __fmul2_rn(e, __fmul2_rn(make_float2(value.x, value.y), c));
            P[i] = pair_of<__half>(w.x, w.y);
        }
        tmem_store8(s + 8 * k, P);
        if (k < 7) check(k + 1, v[(k + 1) & 1], most, steps, x[k & 1]);
    }
    r.l = sum.x + sum.y;
    r.lo = low.x + low.y;
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1) cache_attention_tiles_kernel(const AttParams p) {
    using Sh = TcAttShape<D>;
    constexpr int R = kTcRows;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::kStages + 16];
    __shared__ uint32_t there[Sh::kStages], slot;
    __shared__ int dead;
    uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t* const q_smem = smem;                       // two halves of 128 rows
    uint8_t* const k_smem = q_smem + 2 * Sh::kHalf;
    uint8_t* const v_smem = k_smem + 2 * Sh::kHalf;   // (keys are widened a tile ahead)
    uint8_t* const ring = v_smem + Sh::kHalf;
    uint8_t* const params = ring + Sh::kStages * Sh::kStage;
    int* const first = reinterpret_cast<int*>(params + 2 * Sh::kParam);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(bars), empty = full + 8 * Sh::kStages, k_full = empty + 8 * Sh::kStages, k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 8,
                   s_full = v_empty + 8, p_full = s_full + 16, o_full = p_full + 16, par_full = o_full + 16, q_full = par_full + 16, done = q_full + 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < Sh::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 4);
        mbar_init(v_full, 4), mbar_init(v_empty, 1);
        for (int i = 0; i < 2; ++i) mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, 4), mbar_init(o_full + 8 * i, 1), mbar_init(par_full + 8 * i, 4), mbar_init(k_full + 8 * i, 4), mbar_init(k_empty + 8 * i, 1);
        mbar_init(q_full, 8), mbar_init(done, 1);
        fence_mbar_init();
        dead = 0;
    }
    if (warp == 12) {
        tmem_alloc(smem_u32(&slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_launch();   // only now: a next kernel's blocks could take the columns
    const uint32_t tmem = slot;
    griddep_wait();
    att_units<R>(p, first, kTcThreads);
    const int units = first[p.c.seqs], cta = blockIdx.x;
    const AttShare sh(p, units);
    const int shift = min(p.c.shift, 7), pieces = kAttTile >> shift;
    // Waits: whoever gives up says so and waits for nothing more; the others do as they come to it.
    bool lost = false;
    const auto wait = [&](uint32_t bar, int parity, int code) {
        if (lost) return;
        if (!mbar_wait_warp(bar, parity, p.wait_limit)) {
            lost = true;
            if (lane == 0) *p.err = code, *static_cast<volatile int*>(&dead) = 1;
        }
        if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&dead))) lost = true;
    };

    if (warp == 13) {   // ---- copies tiles in
        int stage = 0, phase = 0;
        long long issued = 0;
        const long long half = D / 2;
        const uint32_t codes = static_cast<uint32_t>(half) << shift, pairs = 4u << shift;
        for (int u = sh.beg; u < sh.end && !lost;) {
            const AttItem it = att_item<R>(p, first, u);
            int t0, t1;
            att_tiles(p, it, sh.beg, sh.end, t0, t1);
            u = it.next;
            const int per = 32 / pieces;   // tiles whose pages the lanes look up at once
            for (int tb = t0; tb < t1 && !lost; tb += per) {
                const int mine = tb + lane / pieces;
                const long long pos = static_cast<long long>(mine) * kAttTile + (lane % pieces << shift);
                int page = -1;
                if (mine < t1 && pos < it.seen) page = page_of(p.c, it.b, pos);
                const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
                for (int i = 0; i < per && tb + i < t1; ++i) {
                    wait(empty + 8 * stage, phase ^ 1, ERR_WAIT_EMPTY);
                    if (lost) break;
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
                        const int at = lane % pieces << shift;
                        const long long in = pos & (p.c.page - 1);
                        const uint32_t dst = smem_u32(ring) + stage * Sh::kStage, bar = full + 8 * stage;
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
        // no copy is in flight when the block ends
        for (long long i = max(0LL, issued - Sh::kStages); i < issued; ++i)
            if (!mbar_wait_warp(full + 8 * static_cast<int>(i % Sh::kStages), static_cast<int>(i / Sh::kStages) & 1, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
    } else if (warp == 12) {   // ---- issues MMAs
        const uint64_t qd = make_sdesc(smem_u32(q_smem), 128), kd = make_sdesc(smem_u32(k_smem), 128), vd = n_major_desc(smem_u32(v_smem), Sh::kBlock);
        int tile = 0, item = 0;   // how many so far
        int turns[2] = {0, 0};    // of P
        const auto scores = [&](int g, int which, bool last) {   // which: of the keys' buffers
            if (lost) return;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint64_t at = static_cast<uint64_t>((k / 4 * Sh::kBlock + k % 4 * 32) >> 4);
                mma_f16(tmem + 128 * g, qd + (g * Sh::kHalf >> 4) + at, kd + (which * Sh::kHalf >> 4) + at, idesc_f16(128, false), k > 0);
            }
            mma_commit_elect(s_full + 8 * g);
            if (last) mma_commit_elect(k_empty + 8 * which);
        };
        for (int u = sh.beg; u < sh.end;) {
            const AttItem it = att_item<R>(p, first, u);
            int t0, t1;
            att_tiles(p, it, sh.beg, sh.end, t0, t1);
            u = it.next;
            if (t0 >= t1) continue;
            const int groups = it.rows - it.row0 > 128 ? 2 : 1;
            wait(q_full, item++ & 1, ERR_WAIT_FULL);
            wait(k_full + 8 * (tile & 1), (tile >> 1) & 1, ERR_WAIT_FULL);
            for (int g = 0; g < groups; ++g) scores(g, tile & 1, g == groups - 1);
            for (int t = t0; t < t1; ++t, ++tile) {
                wait(v_full, tile & 1, ERR_WAIT_FULL);
                for (int g = 0; g < groups; ++g) {
                    wait(p_full + 8 * g, turns[g]++ & 1, ERR_WAIT_ACC);
                    if (lost) continue;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_f16_tmem(tmem + 256 + 128 * g, tmem + 128 * g + 8 * k, vd + (k * 2048 >> 4), idesc_f16(D, true), t > t0 || k > 0);
                    if (g == groups - 1) mma_commit_elect(v_empty);
                    if (t + 1 < t1) {
                        if (g == 0) wait(k_full + 8 * ((tile + 1) & 1), ((tile + 1) >> 1) & 1, ERR_WAIT_FULL);
                        scores(g, (tile + 1) & 1, g == groups - 1);
                    } else {
                        mma_commit_elect(o_full + 8 * g);
                    }
                }
            }
        }
        // no product is under way when the columns are given back
        mma_commit_elect(done);
        if (!mbar_wait_warp(done, 0, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
        tc_fence_before();
    } else if (warp >= 8 && warp < 12) {   // ---- widen codes
        const int mine = threadIdx.x - 256;   // token of the parameters
        const uint32_t kv[2] = {smem_u32(k_smem), smem_u32(v_smem)};
        int stage = 0, phase = 0, tile = 0;
        constexpr int LANES = D / 32, ROWS = 32 / LANES;   // lanes of a token's row, 32 codes each; tokens of a warp at a time
        const int part = lane % LANES, row = lane / LANES;
        const auto widen = [&](const uint8_t* from, uint32_t to) {
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += ROWS) {
                const int tok = (warp - 8) * 32 + row + i0;
                const uint4 w = *reinterpret_cast<const uint4*>(from + tok * (D / 2) + part * 16);
                const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int chunk = 4 * part + i;
                    const uint32_t u = words[i], v = u >> 8;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + chunk / 8 * Sh::kBlock + tok * 128 + ((chunk ^ tok) & 7) * 16), "r"(centred_low(u)),
                                 "r"(centred_high(u)), "r"(centred_low(v)), "r"(centred_high(v))
                                 : "memory");
                }
            }
        };
        for (int u = sh.beg; u < sh.end;) {
            const AttItem it = att_item<R>(p, first, u);
            int t0, t1;
            att_tiles(p, it, sh.beg, sh.end, t0, t1);
            u = it.next;
            for (int t = t0; t < t1; ++t, ++tile) {
                const uint8_t* K = ring + stage * Sh::kStage;
                const uint8_t* V = K + Sh::kCodes;
                wait(full + 8 * stage, phase, ERR_WAIT_FULL);
                wait(k_empty + 8 * (tile & 1), ((tile >> 1) & 1) ^ 1, ERR_WAIT_EMPTY);
                if (!lost) {
                    widen(K, kv[0] + (tile & 1) * Sh::kHalf);
                    uint32_t pk = reinterpret_cast<const uint32_t*>(V + Sh::kCodes)[mine], pv = reinterpret_cast<const uint32_t*>(V + Sh::kCodes + Sh::kPairs)[mine];
                    const bool ok = t * kAttTile + mine < it.seen && ((there[stage] >> (mine >> shift)) & 1);
                    if (!ok) pk = pv = 0;   // what lies there is not looked at
                    const float ks = __uint_as_float(pk << 16) * p.key_scale, vs = __uint_as_float(pv << 16);
                    float* to = reinterpret_cast<float*>(params + (tile & 1) * Sh::kParam) + mine / 16 * 64 + mine % 16 / 2 * 4 + mine % 2;
                    to[0] = ks, to[2] = __fmaf_rn(8.0f, ks, __uint_as_float(pk & 0xFFFF0000u) * p.key_scale);
                    to[32] = vs, to[34] = __fmaf_rn(8.0f, vs, __uint_as_float(pv & 0xFFFF0000u));
                    const uint32_t have = __ballot_sync(0xffffffffu, ok);
                    float most = fmaxf(fabsf(vs), 0.0f);   // (NaN counts for nothing)
#pragma unroll
                    for (int d = 1; d < 32; d *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                    if (lane == 0) {
                        uint32_t* end = reinterpret_cast<uint32_t*>(params + (tile & 1) * Sh::kParam + kAttTile * 16);
                        end[warp - 8] = have, end[4 + warp - 8] = __float_as_uint(most);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(par_full + 8 * (tile & 1)), mbar_arrive(k_full + 8 * (tile & 1));   // (in this order: see the softmax's waits)
                wait(v_empty, (tile & 1) ^ 1, ERR_WAIT_EMPTY);
                if (!lost) widen(V, kv[1]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full), mbar_arrive(empty + 8 * stage);
                if (++stage == Sh::kStages) stage = 0, phase ^= 1;
            }
        }
    } else if (warp < 8) {   // ---- softmax
        const int g = warp >> 2, my = threadIdx.x & 127;
        const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21, s = tmem + quarter + 128 * g, o = tmem + quarter + 256 + 128 * g;
        const long long cap = static_cast<long long>(p.c.width) << p.c.shift;
        int tile = 0, turns = 0, ends = 0, items = 0;
        if (!p.by_item && !p.listed && threadIdx.x == 0) p.desc[cta].last = -1;
        for (int u = sh.beg; u < sh.end;) {
            const AttItem it = att_item<R>(p, first, u);
            int t0, t1;
            att_tiles(p, it, sh.beg, sh.end, t0, t1);
            u = it.next;
            if (t0 >= t1) continue;
            const bool cut = t0 > 0 || t1 < it.tiles;
            const int row = it.row0 + 128 * g + my;
            const bool mine = row < it.rows;
            const long long from = mine ? (it.token0 + row / p.per) * p.q_token + static_cast<long long>(it.head * p.per + row % p.per) * p.q_head : 0;
            TcRow r;
            {   // the row's queries: scaled so that the largest is 2^14 .. 2^15
                float top = 0.0f, sum = 0.0f;
                const auto value = [&](int k) { return mine ? att_value(p.q, from + k, p.type) : 0.0f; };
                const auto eight = [&](int k, float (&f)[8]) {
                    if (mine && p.vec_q) {
                        if (p.type == Y_F16)
                            load8<__half, true>(static_cast<const __half*>(p.q) + from + k, f);
                        else
                            load8<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(p.q) + from + k, f);
                    } else {
#pragma unroll
                        for (int z = 0; z < 8; ++z) f[z] = value(k + z);
                    }
                };
#pragma unroll 4
                for (int k = 0; k < D; k += 8) {
                    float f[8];
                    eight(k, f);
#pragma unroll
                    for (int z = 0; z < 8; ++z) top = max_nan(top, fabsf(f[z]));
                }
                const int e = att_power(top);
                const float up = exp2_int(e);
                const uint32_t to = smem_u32(q_smem) + g * Sh::kHalf + my * 128;
#pragma unroll 4
                for (int k = 0; k < D; k += 8) {
                    float f[8];
                    eight(k, f);
#pragma unroll
                    for (int z = 0; z < 8; ++z) f[z] *= up, sum += f[z];
                    const int chunk = k / 8;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + chunk / 8 * Sh::kBlock + ((chunk ^ my) & 7) * 16), "r"(pair_of<__half>(f[0], f[4])),
                                 "r"(pair_of<__half>(f[1] * 0.0625f, f[5] * 0.0625f)), "r"(pair_of<__half>(f[2], f[6])), "r"(pair_of<__half>(f[3] * 0.0625f, f[7] * 0.0625f))
                                 : "memory");
                }
                // NaN and infinities in a row make all of its scores NaN
                r.a = isfinite(top) ? exp2_int(kAttKeys - e) * p.score_scale : __int_as_float(0x7FC00000);
                r.b = sum;
                r.m = r.l = r.lo = 0.0f, r.c = 0x1p120f, r.fresh = true;
                r.lim = mine ? static_cast<int>(min(max(it.len - it.n + row / p.per + 1, 0LL), cap)) : 0x7FFFFFFF;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            ++items;
            if (128 * g >= it.rows - it.row0) {   // no rows of this half: on to the next, but not so soon that its arrival counts for this one
                tile += t1 - t0;
                wait(q_full, (items - 1) & 1, ERR_WAIT_FULL);
                continue;
            }
            const int all = min(it.seen, __reduce_min_sync(0xffffffffu, r.lim));   // positions that all of the warp's rows see
            for (int t = t0; t < t1; ++t, ++tile) {
                const uint8_t* par = params + (tile & 1) * Sh::kParam;
                const float4* param = reinterpret_cast<const float4*>(par);
                const uint32_t* have = reinterpret_cast<const uint32_t*>(par + kAttTile * 16);
                const float* largest = reinterpret_cast<const float*>(have + 4);
                // A half that had no rows in the items before comes here any number of tiles early, where a phase of par_full long past may have the
                // parity that it waits for.  What keeps it from this tile's parameters until they are there is s_full, which has phases for the half's
                // own tiles only: scores follow all arrivals at k_full, and whoever arrives there has arrived at par_full before.  (Waiting for the
                // scores first: 254 us instead of 247; so for an item's first tile only: 250.)
                wait(par_full + 8 * (tile & 1), (tile >> 1) & 1, ERR_WAIT_FULL);
                wait(s_full + 8 * g, turns++ & 1, ERR_WAIT_ACC);
                if (!lost) {
                    tc_fence_after();
                    const bool masked = (t + 1) * kAttTile > all || (have[0] & have[1] & have[2] & have[3]) != 0xFFFFFFFFu;
                    const float step = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
                    const int ocols = t > t0 ? D : 0;
                    if (masked)
                        tc_tile<true>(r, s, o, ocols, param, have, t * kAttTile, step);
                    else
                        tc_tile<false>(r, s, o, ocols, param, have, t * kAttTile, step);
                    tmem_stored();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * g);
            }
            // ---- the segment's end
            wait(o_full + 8 * g, ends++ & 1, ERR_WAIT_ACC);
            tc_fence_after();
            const float inv = power_ratio(1.0f, r.c), div = r.l == 0.0f ? 0.0f : 1.0f / r.l;   // a row that sees nothing: zeros
            const long long slot_row = (2LL * cta + (t0 == 0)) * R + 128 * g + my;
            const long long at = mine ? (it.token0 + row / p.per) * p.o_token + static_cast<long long>(it.head * p.per + row % p.per) * p.o_head : 0;
            for (int d = 0; d < D && !lost; d += 16) {   // (a block that gives up leaves what it would; its row tiles are described all the same)
                uint32_t x[16];
                __syncwarp();   // (the loads are the whole warp's; what follows is not)
                tmem_ld16(o + d, x);
                tmem_wait_ld(x);
                if (!mine) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float y[8];
#pragma unroll
                    for (int z = 0; z < 8; ++z) {   // column z is dimension (z / 2) + 4 (z % 2), the odd ones 16 times too large
                        const float v = __uint_as_float(x[8 * h + z]) * (z & 2 ? 0.0625f : 1.0f);
                        y[z / 2 + 4 * (z & 1)] = __fmaf_rn(v, inv, r.lo);
                    }
                    const int k = d + 8 * h;
                    if (cut) {
                        float* to = p.part + slot_row * D + k;
                        reinterpret_cast<float4*>(to)[0] = make_float4(y[0], y[1], y[2], y[3]);
                        reinterpret_cast<float4*>(to)[1] = make_float4(y[4], y[5], y[6], y[7]);
                    } else {
#pragma unroll
                        for (int z = 0; z < 8; ++z) y[z] *= div;
                        if (p.type == Y_F16) {
                            __half* to = static_cast<__half*>(p.out) + at + k;
                            p.vec_o ? store8<__half, true>(to, y) : store8<__half, false>(to, y);
                        } else {
                            __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.out) + at + k;
                            p.vec_o ? store8<__nv_bfloat16, true>(to, y) : store8<__nv_bfloat16, false>(to, y);
                        }
                    }
                }
            }
            __syncwarp();
            if (cut && mine) p.stat[2 * slot_row] = r.fresh ? kAttNone : r.m, p.stat[2 * slot_row + 1] = r.l;
            if (t0 == 0 && threadIdx.x == 0 && (p.listed || cut)) p.desc[p.listed ? it.index : cta] = att_described(it, sh, cta, cut);
            tc_fence_before();
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace ptq8

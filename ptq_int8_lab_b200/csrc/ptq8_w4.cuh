// Products of float activations with 4-bit weights that have a scale per group of input features:
//   y[t][c] = sum_g s[c][g] (sum_{k in group g} code[c][k] x[t][k]) + b[c], then the epilogue
// for a few tokens, whose activations stay as they are (f32, f16 or bf16).
//
// A code enters the tensor cores as a normal f16 number around zero (16 times it, for the second code of a byte): masked out of
// a word together with the exponent of 1024, less 1032.  (code + 8 alone, as the subnormal number that it is in a word, is an
// instruction less for two codes, but the tensor cores line the products of a sum up by their operands' exponents, take a
// subnormal number's for 2^-14, and cut what is below: an activation 2^12 times the others cost an output 2^-10 of itself, even
// where its code is zero.  8 tokens, 4096 -> 2 x 8192: 14.9 us, 14.8 so.)  Activations become f16 times a power of two, which
// takes the largest of 128 to 2^14 .. 2^15, those that meet a byte's second code a sixteenth of it: what is within 2^28 (2^24) of
// the largest keeps f16's and bf16's places, and f16's finest step is 2^-38 (2^-34) of it.  f32 ones go in as two f16, the second
// with what the first leaves (22 places, down to that step), in columns beside each other.  A group's sum is f32 in the tensor cores, and
// meets its scale in f32.
//
// A warp has pairs of tiles of 16 weight rows, or shares each with split - 1 others, which take other input features; their sums
// meet in shared memory, in a fixed order.  Weights come by TMA through a ring of the warp's own in shared memory, two
// chunks of 128 features of the 32 rows at a time.  (Bulk copies of single rows, a lane each, run one after another
// in some 20 instructions each: 32 of them took 2 us.)  The activations are brought into the products' order in shared
// memory: once, where they fit there as a whole, else a segment at a time.  Places of the products' inner dimension are
// dealt to a row's bytes so that a group stays within an MMA (four lanes hold VB bytes each: 32, 64 or 128 codes of a row).
// EXACT (outputs of 32 bits): each product of 16 features begins at zero and is added in f32 (45 tokens x 2000, f32: 8.6e-8 from 64 bits).
//
// What it spends its time on (B200, in a graph of calls): one token, 4096 -> 4096, 4.9 us, floor 1.3: latency and launch (8.7 MB at
// 1.8 TB/s, from L2; 5.2 us with weights from DRAM); 8 tokens, 4096 -> 2 x 8192, 15 us, floor 5.5: waits for the weights' and fragments'
// way through shared memory and for the instructions that widen them (issue 53 %), after 3 us in which every block brings the activations
// into order; 45 tokens f32, 2000 -> 1270, 10.1 us: that same start, for three passes of 16 tokens.  Beyond some tens of tokens every
// pass of at most 32 reads and widens all weights again: 512 bf16 tokens, 4096 -> 4096, 127 us where the operations' floor is 11.
// Kernels of four tiles of eight columns spill (up to 282 bytes of stores and 372 of loads), those of one do not.
#pragma once

#include "ptq8_cache.cuh"
#include "ptq8_linear.cuh"
#include "ptq8_rows.cuh"

namespace ptq8 {

constexpr int kW4Warps = 16, kW4Chunk = 128;

struct W4Params {
    const void* x;
    const uint8_t* w;
    const void* s;
    const float* bias;
    void* y;
    size_t ldx, ldw, lds, ldy;   // elements, bytes, elements, elements
    long long rows;
    int k, n, group;             // n: output features
    int gated, x_type, s_type, y_type;
    int vec_x;      // activations at multiples of 16 bytes
    int shift;      // group = 1 << shift, or -1
    long long wait_limit;
    int* err;
    int stall;
};

__device__ __forceinline__ float scale_at(const W4Params& p, size_t at) {
    if (p.s_type == Y_F32) return static_cast<const float*>(p.s)[at];
    if (p.s_type == Y_F16) return __half2float(static_cast<const __half*>(p.s)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p.s)[at]);
}
__device__ __forceinline__ float x_at(const W4Params& p, size_t at) {
    if (p.x_type == Y_F32) return static_cast<const float*>(p.x)[at];
    if (p.x_type == Y_F16) return __half2float(static_cast<const __half*>(p.x)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p.x)[at]);
}

// Any layout, any group: a warp per output feature, four tokens at a time, a lane a byte of weights.
constexpr int kW4AnyTokens = 4;

__global__ void __launch_bounds__(256) linear_w4_any_kernel(const W4Params p) {
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, c = blockIdx.x * 8 + (threadIdx.x >> 5), halves = p.gated ? 2 : 1;
    if (c >= p.n) return;
    for (long long t0 = static_cast<long long>(blockIdx.y) * kW4AnyTokens; t0 < p.rows; t0 += static_cast<long long>(gridDim.y) * kW4AnyTokens) {
        float acc[2][kW4AnyTokens] = {};
        for (int h = 0; h < halves; ++h) {
            const size_t row = static_cast<size_t>(h) * p.n + c;
            for (int byte = lane; byte < (p.k + 1) / 2; byte += 32) {
                const int both = p.w[row * p.ldw + byte];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = 2 * byte + i;
                    if (k >= p.k) break;
                    const int code = ((both >> (4 * i) & 15) ^ 8) - 8;
                    const float w = static_cast<float>(code) * scale_at(p, row * p.lds + k / p.group);
#pragma unroll
                    for (int t = 0; t < kW4AnyTokens; ++t)
                        if (t0 + t < p.rows) acc[h][t] = __fmaf_rn(w, x_at(p, static_cast<size_t>(t0 + t) * p.ldx + k), acc[h][t]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < kW4AnyTokens; ++t) {
            float v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v[h] = acc[h][t];
#pragma unroll
                for (int d = 16; d; d /= 2) v[h] += __shfl_xor_sync(0xffffffffu, v[h], d);
                if (p.bias && h < halves) v[h] += p.bias[static_cast<size_t>(h) * p.n + c];
            }
            if (lane == 0 && t0 + t < p.rows) store_y(p.y, static_cast<size_t>(t0 + t) * p.ldy + c, p.gated ? swiglu(v[0], v[1]) : v[0], p.y_type);
        }
    }
}

__device__ __forceinline__ float w4_scale(uint32_t bits, int type) {
    const float half = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
    const float wide = __uint_as_float(type == Y_F32 ? bits : bits << 16);
    return type == Y_F16 ? half : wide;
}

// One or two tokens: float multiply-adds on weights that go from memory straight to registers, as the few-token products of
// int8 codes have it: a warp owns four weight rows (gated: two gate and two up rows), a lane 32 codes of each at a time, KS
// warps of a block share a row's input features.  A code's byte becomes the float 2^11 + 2^-12 (8 + code) by one byte permutation
// and the code by half of a packed subtraction, exactly; with the packed multiply-adds of T tokens that makes 16 + 4 T
// instructions for 8 codes, and bounds the kernel together with the launch.  Activations are exact floats here.  (All of it times
// 2^-12, by the exponent of those floats: the largest activations times codes stay within f32.)
constexpr int kW4FewWarps = 8, kW4FewRows = 4;

template <typename XT, int MT>
__global__ void __launch_bounds__(32 * kW4FewWarps, 1) linear_w4_few_kernel(const W4Params p, int ks) {
    __shared__ float sums[kW4FewWarps][kW4FewRows * MT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp & (ks - 1), set = warp / ks;
    const int C = p.gated ? kW4FewRows / 2 : kW4FewRows;   // output features of a warp
    const int c0 = (blockIdx.x * (kW4FewWarps / ks) + set) * C, bytes = p.k / 2;   // whole vectors of 16 (the host sees to it)
    const int scale_shift = p.s_type == Y_F32 ? 2 : 1;
    const uint8_t* row[kW4FewRows];
    const char* scales[kW4FewRows];
#pragma unroll
    for (int r = 0; r < kW4FewRows; ++r) {   // rows past the end repeat the last one; their sums are dropped
        const int c = min(c0 + (p.gated ? r & 1 : r), p.n - 1) + (p.gated && r > 1 ? p.n : 0);
        row[r] = p.w + static_cast<size_t>(c) * p.ldw;
        scales[r] = static_cast<const char*>(p.s) + (static_cast<size_t>(c) * p.lds << scale_shift);
    }
    const int strides = (bytes + 511) / 512, s0 = strides * part / ks, s1 = strides * (part + 1) / ks;
    for (int s = s0; s < s1; ++s)   // into L2 while the kernel before this one drains
        if (s * 512 + lane * 16 < bytes)
#pragma unroll
            for (int r = 0; r < kW4FewRows; ++r) asm volatile("prefetch.global.L2 [%0];" ::"l"(row[r] + s * 512 + lane * 16));
    griddep_wait();
    griddep_launch();
    float acc[kW4FewRows][MT] = {};
#pragma unroll 2
    for (int s = s0; s < s1; ++s) {
        const int byte = s * 512 + lane * 16;
        if (byte >= bytes) break;   // (only in the row's last stride)
        uint4 w[kW4FewRows];
        uint32_t scale[kW4FewRows];
        const int at = (p.shift >= 0 ? 2 * byte >> p.shift : 2 * byte / p.group) << scale_shift;
#pragma unroll
        for (int r = 0; r < kW4FewRows; ++r) {
            w[r] = *reinterpret_cast<const uint4*>(row[r] + byte);
            scale[r] = scale_shift == 2 ? *reinterpret_cast<const uint32_t*>(scales[r] + at) : *reinterpret_cast<const unsigned short*>(scales[r] + at);
        }
        float2 sum[kW4FewRows][MT] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // eight codes
            float2 x[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {   // missing tokens repeat the last one; their sums are dropped
                float f[8];
                load8<XT, true>(static_cast<const XT*>(p.x) + min(static_cast<long long>(t), p.rows - 1) * p.ldx + 2 * byte + 8 * i, f);
#pragma unroll
                for (int z = 0; z < 4; ++z) x[t][z] = make_float2(f[2 * z], f[2 * z + 1]);
            }
#pragma unroll
            for (int r = 0; r < kW4FewRows; ++r) {
                const uint32_t v = (&w[r].x)[i] ^ 0x88888888u, even = v & 0x0F0F0F0Fu, odd = v >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float2 c = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(even, 0x45000000u, 0x7440 + z)), __uint_as_float(__byte_perm(odd, 0x45000000u, 0x7440 + z))), both(-0x1.00001p11f));
#pragma unroll
                    for (int t = 0; t < MT; ++t) sum[r][t] = __ffma2_rn(c, x[t][z], sum[r][t]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kW4FewRows; ++r) {
            const float f = w4_scale(scale[r], p.s_type);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = __fmaf_rn(sum[r][t].x + sum[r][t].y, f, acc[r][t]);
        }
    }
    __syncwarp();
    float mine = 0.0f;   // of row lane / MT, token lane % MT
#pragma unroll
    for (int r = 0; r < kW4FewRows; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float v = acc[r][t];
#pragma unroll
            for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
            if (lane == r * MT + t) mine = v;
        }
    if (ks > 1) {
        if (lane < kW4FewRows * MT) sums[warp][lane] = mine;
        __syncthreads();
        if (part == 0 && lane < kW4FewRows * MT)
            for (int i = 1; i < ks; ++i) mine += sums[warp + i][lane];
    }
    const int r = lane / MT, t = lane % MT, c = c0 + (p.gated ? r & 1 : r);
    const bool here = part == 0 && lane < kW4FewRows * MT && c < p.n && t < p.rows;
    mine *= 0x1p12f;
    if (here && p.bias) mine += p.bias[c + (p.gated && r > 1 ? p.n : 0)];
    const float up = __shfl_down_sync(0xffffffffu, mine, 2 * MT);
    if (here && r < C) store_y(p.y, static_cast<size_t>(t) * p.ldy + c, p.gated ? swiglu(mine, up) : mine, p.y_type);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// With every code's sign bit turned a nibble is code + 8.
constexpr uint32_t kW4Turn = 0x88888888u, kW4Low = 0x000F000Fu, kW4High = 0x00F000F0u;
// The code itself (16 times it for the high one) as a normal f16 number: 1024 + 8 + code, less 1032.
__device__ __forceinline__ uint32_t w4_low(uint32_t word) {
    const uint32_t a = mask_or(word, kW4Low, 0x64006400u), b = 0x64086408u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t w4_high(uint32_t word) {
    const uint32_t a = mask_or(word, kW4High, 0x64006400u), b = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <int VB>
struct W4Pieces {
    static constexpr int N = 16 / VB, RUN = 2 * VB;   // of a chunk, that a lane has; consecutive values of one
};

// 32 activations of a lane's token and place of a chunk, as they lie in memory; zeros without a token and behind the row's end.
template <typename XT, int VB>
__device__ __forceinline__ void w4_tokens(uint4 (&x)[2 * sizeof(XT)], const W4Params& p, const char* token, int chunk, int t) {
    constexpr int RUN = W4Pieces<VB>::RUN, PER = 16 / sizeof(XT);   // values of a vector
    if (p.vec_x && (chunk + 1) * kW4Chunk <= p.k) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(XT)); ++i) {
            const int piece = i * PER / RUN, in = i * PER % RUN;
            x[i] = token ? *reinterpret_cast<const uint4*>(token + (chunk * kW4Chunk + piece * 8 * VB + in) * sizeof(XT)) : make_uint4(0, 0, 0, 0);
        }
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(x);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int k = chunk * kW4Chunk + i / RUN * 8 * VB + i % RUN;
            const bool in = token && k + t * RUN < p.k;
            if constexpr (sizeof(XT) == 4) {
                w[i] = in ? reinterpret_cast<const uint32_t*>(token)[k] : 0u;
            } else {
                const uint32_t v = in ? reinterpret_cast<const unsigned short*>(token)[k] : 0u;
                w[i / 2] = i & 1 ? w[i / 2] | v << 16 : v;
            }
        }
    }
}

template <typename XT>
__device__ __forceinline__ float w4_value(const uint32_t* raw, int i) {
    if constexpr (sizeof(XT) == 4) return __uint_as_float(raw[i]);
    if constexpr (__is_same(XT, __half)) return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? raw[i / 2] >> 16 : raw[i / 2])));
    return __uint_as_float(i & 1 ? raw[i / 2] & 0xFFFF0000u : raw[i / 2] << 16);
}

// Outputs are summed in units of 2^11, so that no group's sum of the largest floats, and no power of two that takes one back to
// its size, leaves f32's range.
constexpr int kW4Units = 11;

// They become f16, four to a word of weights (codes 0, 4; 1, 5, which come 16 times too large; 2, 6; 3, 7), times a power of two, at
// to[stride w].  f32: the lanes of even columns take the first f16 of a number, those of odd ones what it leaves.  Beside
// them, for each column, the power of two that its products lack.
template <typename XT, int VB>
__device__ __forceinline__ void w4_fragments(uint4* to, int stride, bool kept, float* beside, const uint4 (&x)[2 * sizeof(XT)], int g, int t) {
    const uint32_t* raw = reinterpret_cast<const uint32_t*>(x);
    float top;
    if constexpr (sizeof(XT) == 4) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max_nan(top, fabsf(__uint_as_float(raw[i])));
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = Vec<XT>::join(m, raw[i]);
        top = __uint_as_float(Vec<XT>::top(m));
    }
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // from -113 for the largest floats on; what is below 2^-100 stays below 2^14, and loses places by that much
    const int e = min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 114);
    const float up = __int_as_float((e + 127) << 23), up16 = up * 0.0625f;
    // a token that is not finite: NaN (as an infinity times a code of zero is)
    if (t == 0) beside[g] = isfinite(top) ? __int_as_float((-kW4Units - e + 127) << 23) : __int_as_float(0x7FC00000);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t b[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const float u = w4_value<XT>(raw, 8 * w + z) * (z & 1 ? up16 : up), v = w4_value<XT>(raw, 8 * w + z + 4) * (z & 1 ? up16 : up);
            b[z] = pair_of<__half>(u, v);
            if constexpr (sizeof(XT) == 4) {
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&b[z]));
                const uint32_t left = pair_of<__half>(u - h.x, v - h.y);
                if (g & 1) b[z] = left;
            }
        }
        if (kept) to[stride * w] = make_uint4(b[0], b[1], b[2], b[3]);
    }
}

constexpr int kW4Threads = 32 * kW4Warps, kW4MostStages = 4, kW4Smem = 224 * 1024, kW4Run = 2, kW4Box = 32 * 64 * kW4Run;   // chunks of a stage; its bytes

template <typename XT, int VB, int NT>
struct W4Shape {
    static constexpr bool kSplit = sizeof(XT) == 4;
    static constexpr int kColumns = kSplit ? 4 : 8, kTokens = NT * kColumns;   // tokens of eight columns; of a pass
    static constexpr int kPieces = W4Pieces<VB>::N;
    static constexpr int kSums = kW4Warps * 2 * NT * 128 * 4;
    // of a chunk; columns: those held (fewer than eight where there are no more)
    static constexpr int frag(int columns) { return NT * 4 * columns * 64; }
    static constexpr int kBeside = NT * 32;
};

// What the host has worked out (quotients by numbers that are known at launch only cost a warp some hundred cycles each).
struct W4Plan {
    int columns;          // of a tile, that hold a token
    int held, segments;   // chunks whose activations shared memory holds: all, or a segment's; how many segments
    int split_log;        // 1 << split_log warps have a pair of tiles
    int pairs, rounds;    // pairs of tiles; how many a warp has, at most
    int stages;           // of a warp
    int passes;           // over the tokens
};

// EXACT (outputs of 32 bits): what the tensor cores cut of a sum goes by its largest term, so each product of 16 features begins at
// zero there and is added in f32.
template <typename XT, int VB, int NT, bool EXACT>
__global__ void __launch_bounds__(kW4Threads, 1) linear_w4_kernel(const W4Params p, const W4Plan plan, const __grid_constant__ CUtensorMap map) {
    using Sh = W4Shape<XT, VB, NT>;
    constexpr int PIECES = Sh::kPieces, WORDS = VB / 4;
    extern __shared__ uint8_t smem_any[];
    uint8_t* smem = smem_any + (-smem_u32(smem_any) & 1023);   // TMA's pattern of 128 bytes goes by the address
    __shared__ __align__(8) uint64_t bars[kW4Warps * kW4MostStages];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // the lane's row of eight: those of the lanes that read together lie in other banks of TMA's pattern
    const int rg = VB == 16 ? (g >> 1) | (g & 1) << 2 : VB == 8 ? (g & 3) << 1 | g >> 2 : g;
    const int part = warp & ((1 << plan.split_log) - 1), slot = warp >> plan.split_log, slots = kW4Warps >> plan.split_log;
    // rows g and g + 8 of a tile: of a gated product a gate and its up row, else two output features
    const int per = p.gated ? 8 : 16, chunks = (p.k + kW4Chunk - 1) / kW4Chunk;
    const int segments = plan.segments, rounds = plan.rounds, passes = plan.passes;
    uint8_t* ring = smem + warp * plan.stages * kW4Box;
    float* sums = reinterpret_cast<float*>(smem + kW4Warps * plan.stages * kW4Box);   // [warp][2][NT][4][32]
    uint4* frag = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(sums) + Sh::kSums);   // [held][NT][4][columns][4]
    float* beside = reinterpret_cast<float*>(frag + plan.held * NT * 16 * plan.columns);   // [held][NT][8]
    const uint32_t full = smem_u32(bars + warp * kW4MostStages);
    if (lane < plan.stages) mbar_init(full + 8 * lane, 1);
    fence_mbar_init();
    __syncwarp();
    // The pair of tiles that the warp has in a round (past the end: the last one's again; its sums are dropped), and its chunks of a segment.
    // Of a gated product rows 8 r + g and 16 + 8 r + g are tile r's gate and up row g, else rows 16 r + g and 16 r + 8 + g two features.
    const auto pair_of = [&](int round) { return min((round * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x)) * slots + slot, plan.pairs - 1); };
    const auto chunk_of = [&](int segment, int i) { const int n = min(plan.held, chunks - segment * plan.held); return segment * plan.held + (n * i >> plan.split_log); };

    // The warp's stages: for each pass, round and segment, its part of the chunks, two at a time.
    struct Cursor {
        int pass, round, segment, chunk, end;
    };
    const auto begin = [&]() { return Cursor{static_cast<int>(blockIdx.y), 0, 0, chunk_of(0, part), chunk_of(0, part + 1)}; };
    const auto settle = [&](Cursor& c) {   // on to the next part that has chunks, where this one has no more; false: there is none
        while (c.chunk >= c.end) {
            if (c.pass >= passes) return false;
            if (++c.segment == segments) {
                c.segment = 0;
                if (++c.round == rounds) {
                    c.round = 0;
                    c.pass += gridDim.y;
                    if (c.pass >= passes) return false;
                }
            }
            c.chunk = chunk_of(c.segment, part), c.end = chunk_of(c.segment, part + 1);
        }
        return true;
    };
    // Weights go plan.stages ahead of the products.
    Cursor ahead = begin();
    int issued = 0, issue_stage = 0, stage = 0, phase = 0;
    bool lost = false;
    const auto issue = [&]() {
        if (!settle(ahead)) return;
        const int row = pair_of(ahead.round) * 2 * per;
        if (elect_one()) {   // what lies outside of the weights comes as zeros, and counts
            const uint32_t bar = full + 8 * issue_stage, to = smem_u32(ring) + issue_stage * kW4Box;
            mbar_expect_tx(bar, kW4Box);
            if (!(p.stall && blockIdx.x == 0 && blockIdx.y == 0 && warp == 0 && issued == 0)) {
                tma_load_2d(to, &map, bar, ahead.chunk * 64, row);
                if (p.gated) tma_load_2d(to + kW4Box / 2, &map, bar, ahead.chunk * 64, p.n + row);
            }
        }
        __syncwarp();
        ++issued;
        if (++issue_stage == plan.stages) issue_stage = 0;
        ahead.chunk += kW4Run;
    };
    const int scale_shift = p.s_type == Y_F32 ? 2 : 1, scale_pitch = static_cast<int>(p.lds) << scale_shift;   // (the host keeps it an int)
    // into L2 while the kernel before this one drains: what the first stages load
    if (elect_one()) {
        const int row = pair_of(0) * 2 * per;
        for (int c = ahead.chunk; c < min(ahead.end, ahead.chunk + kW4Run * plan.stages); c += kW4Run)
            for (int h = 0; h < (p.gated ? 2 : 1); ++h)
                asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(&map)), "r"(c * 64), "r"(row + h * p.n) : "memory");
    }
    __syncwarp();
    griddep_wait();
    griddep_launch();
    bool started = false;
    for (int pass = blockIdx.y; pass < passes; pass += gridDim.y) {
        const long long t0 = static_cast<long long>(pass) * Sh::kTokens;
        for (int round = 0; round < rounds; ++round) {
            float2 acc[2][NT][2] = {};   // [tile][..][row g or g + 8]: columns 2 t, 2 t + 1
            const char* scales[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int c = min((2 * pair_of(round) + (h >> 1)) * per + rg + (p.gated ? 0 : 8 * (h & 1)), p.n - 1) + (p.gated ? (h & 1) * p.n : 0);
                scales[h] = static_cast<const char*>(p.s) + static_cast<long long>(c) * scale_pitch;
            }
            for (int segment = 0; segment < segments; ++segment) {
                if (segments > 1 || round == 0) {   // the activations of its chunks
                    if (round || segment || pass != static_cast<int>(blockIdx.y)) __syncthreads();   // those before are read
                    const int first = segment * plan.held, count = min(plan.held, chunks - first) * NT;
                    const auto token_at = [&](int i) {
                        const long long token = t0 + i % NT * Sh::kColumns + (Sh::kSplit ? g >> 1 : g);
                        return token < p.rows ? static_cast<const char*>(p.x) + (static_cast<size_t>(token) * p.ldx + t * W4Pieces<VB>::RUN) * sizeof(XT) : nullptr;
                    };
                    for (int i = warp; i < count; i += kW4Warps) {
                        uint4 x[2 * sizeof(XT)];
                        w4_tokens<XT, VB>(x, p, token_at(i), first + i / NT, t);
                        if (!started) {   // (behind the first activations' loads)
                            started = true;
                            for (int i = 0; i < plan.stages; ++i) issue();
                        }
                        w4_fragments<XT, VB>(frag + i * 16 * plan.columns + lane, 4 * plan.columns, g < plan.columns, beside + i * 8, x, g, t);
                    }
                    if (!started) {   // a warp without a share of the activations
                        started = true;
                        for (int i = 0; i < plan.stages; ++i) issue();
                    }
                    __syncthreads();
                }
                const int end = chunk_of(segment, part + 1);
                for (int c0 = chunk_of(segment, part); c0 < end; c0 += kW4Run) {
                    const int n = min(kW4Run, end - c0);
                    // Scales as bits: a conversion here would wait for the load.  [chunk][h]: row g + 8 (h % 2) of tile h / 2.  (Loaded a stage
                    // ahead they took the registers that keep the products' operands out of local memory: 16.0 us instead of 15.8.)
                    uint32_t scale[kW4Run][4];
#pragma unroll
                    for (int j = 0; j < kW4Run; ++j) {
                        const int k = min((c0 + j) * kW4Chunk + min(t, PIECES - 1) * 8 * VB, p.k - 1), at = (p.shift >= 0 ? k >> p.shift : k / p.group) << scale_shift;
                        if (scale_shift == 2) {
#pragma unroll
                            for (int h = 0; h < 4; ++h) scale[j][h] = *reinterpret_cast<const uint32_t*>(scales[h] + at);
                        } else {
#pragma unroll
                            for (int h = 0; h < 4; ++h) scale[j][h] = *reinterpret_cast<const unsigned short*>(scales[h] + at);
                        }
                    }
                    // (a warp that gives up goes on without loads, so that it meets the others at the barriers)
                    if (!lost && !mbar_wait_warp(full + 8 * stage, phase, p.wait_limit)) {
                        lost = true;
                        if (lane == 0) *p.err = ERR_WAIT_FULL;
                    }
                    const uint8_t* tile = ring + stage * kW4Box + rg * 128;
                    // (a lane of a column that holds no token takes the last one's: what it adds to is not used)
                    const uint4* b_at = frag + (c0 - segment * plan.held) * NT * 16 * plan.columns + 4 * min(g, plan.columns - 1) + t;
                    const float* beside_at = beside + (c0 - segment * plan.held) * NT * 8 + 2 * t;
#pragma unroll
                    for (int j = 0; j < kW4Run; ++j) {
                        if (j >= n) break;
                        uint32_t weights[4][4];
#pragma unroll
                        for (int h = 0; h < 4; ++h)
#pragma unroll
                            for (int i = 0; i < PIECES; ++i) {
                                // 16 bytes of a row lie at their place ^ the row's number % 8
                                const int row = p.gated ? 16 * (h & 1) + 8 * (h >> 1) : 8 * h, at = j * 64 + i * 4 * VB + t * VB;
                                const uint8_t* from = tile + row * 128 + (at ^ (rg << 4));
                                uint32_t* w = &weights[h][i * WORDS];
                                if constexpr (VB == 16) {
                                    const uint4 v = *reinterpret_cast<const uint4*>(from);
                                    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                                } else if constexpr (VB == 8) {
                                    const uint2 v = *reinterpret_cast<const uint2*>(from);
                                    w[0] = v.x, w[1] = v.y;
                                } else {
                                    w[0] = *reinterpret_cast<const uint32_t*>(from);
                                }
                            }
                        float2 lack[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) lack[nt] = *reinterpret_cast<const float2*>(beside_at + (j * NT + nt) * 8);
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            float sum[2][NT][4] = {};
#pragma unroll
                            for (int w = i * WORDS; w < (i + 1) * WORDS; ++w) {
                                uint4 b[NT];
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) b[nt] = b_at[((j * NT + nt) * 4 + w) * 4 * plan.columns];
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    const uint32_t u = weights[2 * r][w] ^ kW4Turn, v = weights[2 * r + 1][w] ^ kW4Turn, u8 = u >> 8, v8 = v >> 8;
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) {
                                        if constexpr (EXACT) {
                                            float one[4] = {}, two[4] = {};
                                            mma_f16(one, w4_low(u), w4_low(v), w4_high(u), w4_high(v), b[nt].x, b[nt].y);
                                            mma_f16(two, w4_low(u8), w4_low(v8), w4_high(u8), w4_high(v8), b[nt].z, b[nt].w);
#pragma unroll
                                            for (int z = 0; z < 4; ++z) sum[r][nt][z] += one[z] + two[z];
                                        } else {
                                            mma_f16(sum[r][nt], w4_low(u), w4_low(v), w4_high(u), w4_high(v), b[nt].x, b[nt].y);
                                            mma_f16(sum[r][nt], w4_low(u8), w4_low(v8), w4_high(u8), w4_high(v8), b[nt].z, b[nt].w);
                                        }
                                    }
                                }
                            }
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const float2 s = both(w4_scale(PIECES == 1 ? scale[j][h] : __shfl_sync(0xffffffffu, scale[j][h], (lane & 28) + i), p.s_type));
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const float* x = sum[h >> 1][nt] + 2 * (h & 1);
                                    acc[h >> 1][nt][h & 1] = __ffma2_rn(__fmul2_rn(make_float2(x[0], x[1]), lack[nt]), s, acc[h >> 1][nt][h & 1]);
                                }
                            }
                        }
                    }
                    __syncwarp();   // the stage is read
                    if (++stage == plan.stages) stage = 0, phase ^= 1;
                    if (!lost) issue();
                }
            }
            // The parts' sums meet in the tile's first warp, in their order.
            if (plan.split_log) {
                if (round || pass != static_cast<int>(blockIdx.y)) __syncthreads();   // those before are read
                float2* mine = reinterpret_cast<float2*>(sums) + warp * 4 * NT * 32 + lane;
                if (part)
#pragma unroll
                    for (int i = 0; i < 4 * NT; ++i) mine[32 * i] = acc[i / (2 * NT)][i / 2 % NT][i % 2];
                __syncthreads();
                if (part == 0)
                    for (int w = 1; w < 1 << plan.split_log; ++w)
#pragma unroll
                        for (int i = 0; i < 4 * NT; ++i) {
                            float2& x = acc[i / (2 * NT)][i / 2 % NT][i % 2];
                            x = __fadd2_rn(x, mine[(w * 4 * NT + i) * 32]);
                        }
            }
            const int pair = (round * gridDim.x + blockIdx.x) * slots + slot;
            if (part || pair >= plan.pairs) continue;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int col = 0; col < (Sh::kSplit ? 1 : 2); ++col) {
                        const long long token = t0 + nt * Sh::kColumns + (Sh::kSplit ? t : 2 * t + col);
                        if (token >= p.rows) continue;
                        float v[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) v[h] = (Sh::kSplit ? acc[r][nt][h].x + acc[r][nt][h].y : col ? acc[r][nt][h].y : acc[r][nt][h].x) * (1 << kW4Units);
                        const size_t row = static_cast<size_t>(token) * p.ldy;
                        if (p.gated) {
                            const int c = (2 * pair + r) * 8 + rg;
                            if (c < p.n) store_y(p.y, row + c, swiglu(v[0] + (p.bias ? p.bias[c] : 0.0f), v[1] + (p.bias ? p.bias[p.n + c] : 0.0f)), p.y_type);
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (const int c = (2 * pair + r) * 16 + rg + 8 * h; c < p.n) store_y(p.y, row + c, v[h] + (p.bias ? p.bias[c] : 0.0f), p.y_type);
                        }
                    }
        }
    }
    if (lost)   // no copy is in flight when the block ends
        for (int i = max(0, issued - plan.stages); i < issued; ++i)
            if (!mbar_wait_warp(full + 8 * (i % plan.stages), (i / plan.stages) & 1, p.wait_limit) && lane == 0) *p.err = ERR_DRAIN;
}

}  // namespace ptq8

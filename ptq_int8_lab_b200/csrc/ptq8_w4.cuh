// Products of float activations with 4-bit weights that have a scale per group of input features:
//   y[t][c] = sum_g s[c][g] (sum_{k in group g} code[c][k] x[t][k]) + b[c], then the epilogue
// for a few tokens, whose activations stay as they are (f32, f16 or bf16).
//
// A code enters the tensor cores as it lies in memory: code + 8, masked out of a word, is as f16 the subnormal number
// (code + 8) * 2^-24 (or 16 times it, for the second code of a byte), exact and without a conversion; the 8 leaves with
// a product of a constant row, which starts the sum at -8 sum(x).  Activations become f16 times a power of two, which
// takes the largest of 128 to 2^14 .. 2^15: what is less than 2^28 below it keeps all places of bf16 and f16.  f32 ones
// go in as two f16, the second with what the first leaves (22 places), in columns beside each other.  A group's sum is
// f32 in the tensor cores, and meets its scale in f32.
//
// A warp owns 16 RT weight rows and a part of the input features, a lane 4, 8 or 16 bytes of two of them at a time; the
// eight warps of a block have the same rows, and meet at the end in shared memory, in a fixed order.  Places of the
// products' inner dimension are dealt to a row's bytes so that a group stays within an MMA (four lanes hold VB bytes
// each: 32, 64 or 128 codes of a row).
#pragma once

#include "ptq8_cache.cuh"
#include "ptq8_linear.cuh"

namespace ptq8 {

constexpr int kW4Warps = 8, kW4Chunk = 128;

struct W4Params {
    const void* x;
    const uint8_t* w;
    const void* s;
    const float* bias;
    void* y;
    size_t ldx, ldw, lds, ldy;   // elements, bytes, elements, elements
    long long rows;
    int k, n, group;             // n: output features
    int gated, x_type, s_type, y_type, vec_x;
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

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The nibble's sign bit turned: code + 8 as an unsigned number, as f16 times 2^-24 (16 * 2^-24 for the high one).
constexpr uint32_t kW4Low = 0x000F000Fu, kW4High = 0x00F000F0u, kW4FlipLow = 0x00080008u, kW4FlipHigh = 0x00800080u;
// -8 * 2^-24 and -128 * 2^-24
constexpr uint32_t kW4ShiftLow = 0x80088008u, kW4ShiftHigh = 0x80808080u;

// A lane's part of a chunk: for each of 128 / (8 VB) pieces VB bytes of 2 RT rows; their scales, piece min(t, last)'s.
template <int VB, int RT>
struct W4Load {
    static constexpr int PIECES = 16 / VB;
    uint32_t w[RT][2][4];
    float s[RT][2];
};

template <int VB, int RT>
__device__ __forceinline__ void w4_load(W4Load<VB, RT>& l, const W4Params& p, const uint8_t* const (&row)[RT][2], const size_t (&srow)[RT][2], int chunk, int t) {
    constexpr int PIECES = W4Load<VB, RT>::PIECES;
    const int bytes = (p.k + 1) / 2, at = chunk * 64 + t * VB;
    const int k = min(chunk * kW4Chunk + min(t, PIECES - 1) * 8 * VB, p.k - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l.s[r][h] = scale_at(p, srow[r][h] + k / p.group);
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int from = at + i * 4 * VB;
                uint32_t* w = &l.w[r][h][i * (VB / 4)];
                if (from + VB <= bytes) {
                    if constexpr (VB == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(row[r][h] + from);
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    } else if constexpr (VB == 8) {
                        const uint2 v = *reinterpret_cast<const uint2*>(row[r][h] + from);
                        w[0] = v.x, w[1] = v.y;
                    } else {
                        w[0] = *reinterpret_cast<const uint32_t*>(row[r][h] + from);
                    }
                } else {   // the row's end: byte by byte (what is behind it meets zeros)
#pragma unroll
                    for (int j = 0; j < VB / 4; ++j) w[j] = join4(row[r][h] + from + 4 * j, min(4, bytes - from - 4 * j));
                }
            }
        }
}

// 32 activations of a lane's token, of its places of a chunk, as f32 (zeros behind the row's end or without a token).
template <typename XT, int VB>
__device__ __forceinline__ void w4_tokens(const W4Params& p, float (&f)[32], long long token, int chunk, int t) {
    constexpr int PIECES = 16 / VB, RUN = 2 * VB;   // consecutive values of a piece
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int k0 = chunk * kW4Chunk + i * 8 * VB + t * RUN;
#pragma unroll
        for (int j = 0; j < RUN / 8; ++j) {
            const int k = k0 + 8 * j;
            float e[8];
            if (token >= 0 && p.vec_x && k + 8 <= p.k) {
                load8<XT, true>(static_cast<const XT*>(p.x) + static_cast<size_t>(token) * p.ldx + k, e);
            } else {
#pragma unroll
                for (int z = 0; z < 8; ++z) e[z] = token >= 0 && k + z < p.k ? static_cast<float>(static_cast<const XT*>(p.x)[static_cast<size_t>(token) * p.ldx + k + z]) : 0.0f;
            }
#pragma unroll
            for (int z = 0; z < 8; ++z) f[i * RUN + 8 * j + z] = e[z];
        }
    }
}

// Their f16 as the products want them, four to a word of weights (codes 0, 4; 1, 5, which are 16 times too large; 2, 6; 3, 7),
// and the power of two that their products with code * 2^-24 lack.  SPLIT: a lane of an odd column takes what the even
// column's f16 leave, times 2^11.
template <bool SPLIT>
__device__ __forceinline__ float w4_fragments(uint32_t (&b)[4][4], const float (&f)[32], bool rest) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max_nan(top, fabsf(f[i]));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100);
    const float up = __int_as_float((e + 127) << 23);
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        v[i] = f[i] * up;
        if (SPLIT) {
            const float left = (v[i] - __half2float(__float2half_rn(v[i]))) * 2048.0f;
            if (rest) v[i] = left;
        }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float* x = v + 8 * w;
        b[w][0] = pair_of<__half>(x[0], x[4]);
        b[w][1] = pair_of<__half>(x[1] * 0.0625f, x[5] * 0.0625f);
        b[w][2] = pair_of<__half>(x[2], x[6]);
        b[w][3] = pair_of<__half>(x[3] * 0.0625f, x[7] * 0.0625f);
    }
    // a token that is not finite: NaN (as an infinity times a code of zero is)
    return isfinite(top) ? __int_as_float((24 - e + 127) << 23) : __int_as_float(0x7FC00000);
}

template <typename XT, int VB, int RT, int NT>
__global__ void __launch_bounds__(32 * kW4Warps) linear_w4_kernel(const W4Params p) {
    constexpr bool SPLIT = sizeof(XT) == 4;
    constexpr int TOKENS = NT * (SPLIT ? 4 : 8), PIECES = 16 / VB, WORDS = VB / 4;
    extern __shared__ float sums[];   // [warp][RT][NT][4][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // rows g and g + 8 of a tile: of a gated product a gate and its up row, else two output features
    const int per = p.gated ? 8 : 16, c0 = blockIdx.x * per * RT;
    const uint8_t* row[RT][2];
    size_t srow[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // rows past the end repeat the last one; their sums are dropped
            const int c = min(c0 + r * per + g + (p.gated ? 0 : 8 * h), p.n - 1);
            const size_t at = static_cast<size_t>(c) + (p.gated ? static_cast<size_t>(h) * p.n : 0);
            row[r][h] = p.w + at * p.ldw;
            srow[r][h] = at * p.lds;
        }
    const int chunks = (p.k + kW4Chunk - 1) / kW4Chunk, beg = chunks * warp / kW4Warps, end = chunks * (warp + 1) / kW4Warps;
    griddep_launch();
    griddep_wait();
    for (long long t0 = static_cast<long long>(blockIdx.y) * TOKENS; t0 < p.rows; t0 += static_cast<long long>(gridDim.y) * TOKENS) {
        float acc[RT][NT][4] = {};
        W4Load<VB, RT> cur, next;
        if (beg < end) w4_load(next, p, row, srow, beg, t);
        for (int chunk = beg; chunk < end; ++chunk) {
            cur = next;
            if (chunk + 1 < end) w4_load(next, p, row, srow, chunk + 1, t);
            uint32_t b[NT][4][4];
            float lack[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const long long token = t0 + nt * (TOKENS / NT) + (SPLIT ? g >> 1 : g);
                float f[32];
                w4_tokens<XT, VB>(p, f, token < p.rows ? token : -1, chunk, t);
                const float l = w4_fragments<SPLIT>(b[nt], f, g & 1);
                lack[nt][0] = __shfl_sync(0xffffffffu, l, 8 * t);
                lack[nt][1] = __shfl_sync(0xffffffffu, l, 8 * t + 4);
            }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                float part[RT][NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float shift[4] = {};
#pragma unroll
                    for (int w = i * WORDS; w < (i + 1) * WORDS; ++w) {
                        mma_f16(shift, kW4ShiftLow, kW4ShiftLow, kW4ShiftHigh, kW4ShiftHigh, b[nt][w][0], b[nt][w][1]);
                        mma_f16(shift, kW4ShiftLow, kW4ShiftLow, kW4ShiftHigh, kW4ShiftHigh, b[nt][w][2], b[nt][w][3]);
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int z = 0; z < 4; ++z) part[r][nt][z] = shift[z];
                }
#pragma unroll
                for (int w = i * WORDS; w < (i + 1) * WORDS; ++w)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        uint32_t u = cur.w[r][0][w], v = cur.w[r][1][w];
#pragma unroll
                        for (int z = 0; z < 4; z += 2) {
                            const uint32_t a0 = (u & kW4Low) ^ kW4FlipLow, a1 = (v & kW4Low) ^ kW4FlipLow, a2 = (u & kW4High) ^ kW4FlipHigh, a3 = (v & kW4High) ^ kW4FlipHigh;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_f16(part[r][nt], a0, a1, a2, a3, b[nt][w][z], b[nt][w][z + 1]);
                            u >>= 8, v >>= 8;
                        }
                    }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    float s[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[h] = PIECES == 1 ? cur.s[r][h] : __shfl_sync(0xffffffffu, cur.s[r][h], (lane & 28) + i);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int z = 0; z < 4; ++z) acc[r][nt][z] = __fmaf_rn(part[r][nt][z] * lack[nt][z & 1], s[z >> 1], acc[r][nt][z]);
                }
            }
        }
        // the warps' sums meet, in their order; lane's z: row g + 8 (z / 2), column 2 t + z % 2
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int z = 0; z < 4; ++z) sums[((warp * RT + r) * NT + nt) * 128 + z * 32 + lane] = acc[r][nt][z];
        __syncthreads();
        constexpr int COLUMNS = SPLIT ? 4 : 8;   // tokens of a tile
        for (int i = threadIdx.x; i < RT * NT * COLUMNS * per; i += 32 * kW4Warps) {
            const int in = i % per, r = i / per % RT, col = i / (per * RT) % COLUMNS, nt = i / (per * RT * COLUMNS);
            const int c = c0 + r * per + in;
            const long long token = t0 + nt * COLUMNS + col;
            if (c >= p.n || token >= p.rows) continue;
            const auto sum = [&](int tile_row) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kW4Warps; ++w) {
                    const float* at = sums + ((w * RT + r) * NT + nt) * 128;
                    if (SPLIT) {   // columns 2 col and 2 col + 1
                        const int l = (tile_row & 7) * 4 + col, z = tile_row >> 3 << 1;
                        v += __fmaf_rn(at[(z + 1) * 32 + l], 1.0f / 2048.0f, at[z * 32 + l]);
                    } else {
                        v += at[((tile_row >> 3 << 1) + (col & 1)) * 32 + (tile_row & 7) * 4 + (col >> 1)];
                    }
                }
                return v;
            };
            float v = sum(in);
            if (p.bias) v += p.bias[c];
            if (p.gated) {
                float u = sum(in + 8);
                if (p.bias) u += p.bias[p.n + c];
                v = swiglu(v, u);
            }
            store_y(p.y, static_cast<size_t>(token) * p.ldy + c, v, p.y_type);
        }
        __syncthreads();
    }
}

}  // namespace ptq8

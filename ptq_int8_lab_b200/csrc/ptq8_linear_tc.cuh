// The tensor-core product: tcgen05 kind::i8 with the weights as the M operand.
//
// Output channels are the 128 rows (lanes) of an accumulator and tokens its columns, for every
// number of tokens: a single token pads the 16-column minimum instead of 128 rows, one weight
// tile layout serves all variants, and the epilogue's lanes hold consecutive channels, so that
// plain stores of a warp are consecutive bytes of y whatever y's pitch and alignment.
//
//   CG 2: two CTAs share a tile of 256 channels (cta_group::2); each loads its 128 weight rows
//         and half of the tokens' rows.
//   S > 1 (CG 1): a cluster of S CTAs splits the sum over k; each sends the int32 partial sums
//         of 1/S of the tokens to the CTA that finishes them.  Integer sums: the order of
//         arrival changes nothing.
//   GATED: two accumulators per tile, gate and up channels, joined in the epilogue.
//   W4: weights arrive packed; eight or sixteen warps widen them as 16 times the code (the nibble moved to
//       its byte's high half: no sign extension; the epilogue takes the factor out) and write them to TMEM,
//       from where the MMA takes its M operand.  A thread owns a channel, which is a TMEM lane.  Through
//       shared memory the same took twice the time: writing the widened tile and the MMA's reads of it
//       filled shared memory's bandwidth.
//
// What bounds it (B200; device time in a graph, operands from DRAM):
//   many tokens        4096 x 4096 x 8192 int8 86 us: 3.2 POP/s, the tensor pipe active 89 % of the time, at
//                      the clock that the power limit leaves (int4 90 us; gated 90 and 102 us: two weight tiles
//                      to one of tokens, bound by the 64 bytes a cycle that an SM draws from L2)
//   hundreds           512 x 4096 x 4096 11 us: again L2 to SM, and too few tiles to share them more
//   few                16 x 4096 x 4096 6.5 us: latency (set-up 1, first bytes 1, partial sums 0.7 us), then an MMA
//                      of 16 columns, which takes 55 to 75 cycles instead of 8
//
// Warps: 0 TMA producer, 1 MMA issuer, 2 TMEM and the groups' tile list, 4.. epilogue, then
// (W4) the unpackers.  Waits for data are bounded.  The TMEM allocation and the cluster's barriers have no limit to give;
// they end because what they wait for does: columns are held by kernels that need nothing more of this SM (each lets its
// successor start only once it holds its own), and every thread of a cluster reaches its barriers.
#pragma once

#include "ptq8_linear.cuh"

namespace ptq8 {

enum : int { ERR_WAIT_UNPACK = 5, ERR_WAIT_PARTIAL = 6 };

constexpr int kMaxLinStages = 12;
constexpr long long kLandCycles = 200000;   // about 0.1 ms: far more than a copy to a peer takes
constexpr int kBand = 8;   // token tiles per band of the tile order: a band's operands stay in L2

struct TcParams {
    LinearParams l;
    int kblocks;       // stages of input features: KD blocks of 128
    int stages;
    int split;         // S
    int list_bytes;    // shared memory of the groups' tile list
    int ctiles;        // channel tiles
    uint32_t tmem_cols;
    int acc_bufs;
    long long wait_limit;
    int* err;
    int stall;         // failure test: the first load is announced but not issued
};

template <int CG, int TN, bool W4, bool GATED>
struct TcShape {
    static constexpr int H = GATED ? 2 : 1;
    static constexpr int XR = TN / CG;                     // token rows loaded by one CTA
    // Blocks of 128 input features in a stage: two where one leaves the MMA warp's wait uncovered (4096 x 4096
    // x 8192: 121 -> 99 us; elsewhere loads bound it, and two only make it wait for more).
    static constexpr int KD = CG == 2 && TN == 128 && !W4 && !GATED ? 2 : 1;
    static constexpr int kW = KD * H * 128 * (W4 ? 64 : 128);   // bytes of the weights' rows in a stage
    static constexpr int kXBlock = XR * 128;
    static constexpr int kX = KD * kXBlock;
    static constexpr int kStage = kW + kX;
    static constexpr int kEpi = TN >= 128 ? 8 : 4;          // epilogue warps
    static constexpr int kCW = TN / (kEpi / 4);            // accumulator columns of one warp
    static constexpr int kCols = H * TN;                   // accumulator columns of a tile
    static constexpr int kACols = 32 * H;                  // W4: columns of an operand tile
    // CTAs that share an SM (the next launch's, too: its set-up then overlaps this one's end)
    static constexpr int kPerSm = TN <= (W4 && GATED ? 32 : 64) ? 2 : 1;
    static constexpr int kColumns = 512 / kPerSm;          // of TMEM
    static constexpr int kUnpack = !W4 ? 0 : kPerSm == 2 ? 8 : 16;   // unpacking warps
    static constexpr int kTurns = W4 ? kUnpack / (4 * H) : 1;   // sets of them that take turns at the blocks
    // Two accumulators where TMEM holds them.  With int4 weights the operand tiles have half of it (what two
    // accumulators leave, where CTAs share an SM): they hide the way from the MMAs' release of a tile to its
    // next use.  4096 x 4096 x 4096 gated: 99 us with one accumulator and four operand tiles, 150 us with
    // tiles of 96 tokens, two and two.
    static constexpr int kAccBufs = 2 * kCols > (W4 ? (kPerSm == 2 ? kColumns - kACols : 256) : kColumns) ? 1 : 2;
    static constexpr int kABufs = !W4 ? 0 : kPerSm == 2 ? (kColumns - 2 * kCols) / kACols / kTurns * kTurns : 256 / kACols;
    static constexpr int kACol0 = kPerSm == 2 ? 2 * kCols : 256;     // W4: first column of the operand tiles
    static constexpr int kThreads = 128 + 32 * (kEpi + kUnpack);
    static_assert(!W4 || (kABufs >= 2 && kABufs <= 8 && kABufs % kTurns == 0), "operand tiles");
};

// ---- cluster-wide pieces

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// A relaxed arrival where no data of the thread has to be seen by the peers (a releasing one first waits for its
// stores): barrier set-up, which fence.mbarrier_init orders, and the end of a split tile.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Brings a box of the weights into L2.  Harmless where an earlier kernel of the stream still writes it: L2 is
// where both meet, and the copies that read it come after the wait for that kernel.
__device__ __forceinline__ void prefetch_3d(const CUtensorMap* m, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(m)),
                 "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// Arrive on a barrier of any CTA of the cluster (address from mapa, or of the own CTA) without release: what it orders are
// the thread's tcgen05 accesses, completed by tcgen05.wait, ordered before the arrival by tcgen05.fence::before_thread_sync
// and, at the waiting side, by tcgen05.fence::after_thread_sync.  No data that other instructions wrote may depend on it.
// (With .release.cluster the unpackers took over 1000 cycles a block.)
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Shared-memory accesses by address: the compiler would keep loads through a pointer behind every store to y, which
// it has to think may overlap.
__device__ __forceinline__ int lds32(uint32_t a) {
    int v;
    asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float4 lds128f(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

// Copy from the own shared memory to a CTA's of the cluster; its barrier there counts the bytes.
__device__ __forceinline__ void copy_to_peer(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "r"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <int CG>
__device__ __forceinline__ void load_rows_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
            : "memory");
    else
        tma_load_2d(dst, m, bar, c0, c1);
}
template <int CG>
__device__ __forceinline__ void load_rows_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
            "r"(c1), "r"(c2)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
            "r"(c1), "r"(c2)
            : "memory");
}

// One block of 128 input features: the H tiles' four K slices each (D columns d and d + step), then the
// commit that releases the block -- in one asm block with one election, and descriptors advanced in their
// low words only (the start address, 14 bits that never carry inside shared memory): with an election per
// K chunk and 64-bit adds the issuing warp, not the tensor core, set the pace.
// M operand: shared-memory descriptor (a K slice of 32 codes is 2 units of 16 bytes, the second tile 1024
// units further), or TMEM (8 columns, 32 columns further).
#define PTQ8_MMA(G, D, A, P) "@e tcgen05.mma.cta_group::" G ".kind::i8 [" D "], " A ", B, %5, " P ";\n\t"
#define PTQ8_S(G, D, AO, BO, P)                                                                             \
    "add.u32 ta, %2, " AO ";\n\tadd.u32 tb, %3, " BO ";\n\tmov.b64 A, {ta, %4};\n\tmov.b64 B, {tb, %4};\n\t" \
    PTQ8_MMA(G, D, "A", P)
#define PTQ8_T(G, D, AO, BO, P)                                                                             \
    "add.u32 ta, %2, " AO ";\n\tadd.u32 tb, %3, " BO ";\n\tmov.b64 B, {tb, %4};\n\t" PTQ8_MMA(G, D, "[ta]", P)
#define PTQ8_S4(G) PTQ8_S(G, "%0", "0", "0", "p") PTQ8_S(G, "%0", "2", "2", "1") PTQ8_S(G, "%0", "4", "4", "1") PTQ8_S(G, "%0", "6", "6", "1")
#define PTQ8_S8(G) PTQ8_S4(G) PTQ8_S(G, "%1", "1024", "0", "p") PTQ8_S(G, "%1", "1026", "2", "1") PTQ8_S(G, "%1", "1028", "4", "1") PTQ8_S(G, "%1", "1030", "6", "1")
#define PTQ8_T4(G) PTQ8_T(G, "%0", "0", "0", "p") PTQ8_T(G, "%0", "8", "2", "1") PTQ8_T(G, "%0", "16", "4", "1") PTQ8_T(G, "%0", "24", "6", "1")
#define PTQ8_T8(G) PTQ8_T4(G) PTQ8_T(G, "%1", "32", "0", "p") PTQ8_T(G, "%1", "40", "2", "1") PTQ8_T(G, "%1", "48", "4", "1") PTQ8_T(G, "%1", "56", "6", "1")
#define PTQ8_D(G, AO, BO)                                                                                   \
    "add.u32 ta, %2, " AO ";\n\tadd.u32 tb, %8, " BO ";\n\tmov.b64 A, {ta, %4};\n\tmov.b64 B, {tb, %4};\n\t" \
    PTQ8_MMA(G, "%0", "A", "1")
#define PTQ8_D8(G) PTQ8_S4(G) PTQ8_D(G, "1024", "0") PTQ8_D(G, "1026", "2") PTQ8_D(G, "1028", "4") PTQ8_D(G, "1030", "6")
#define PTQ8_COMMIT1 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t}\n"
#define PTQ8_COMMIT2                                                                                        \
    "mov.u16 m, 3;\n\t@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%7], m;\n\t}\n"
#define PTQ8_BLOCK(BODY)                                                                                    \
    asm volatile(                                                                                           \
        "{\n\t.reg .pred e, p;\n\t.reg .b64 A, B;\n\t.reg .b32 ta, tb;\n\t.reg .b16 m;\n\t"                  \
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %6, 0;\n\t" BODY ::"r"(d), "r"(d + step), "r"(a),     \
        "r"(b), "r"(hi), "r"(idesc), "r"(acc), "r"(bar), "r"(b2)                                            \
        : "memory")

// a: TMEM address (TMEM_A) or low word of the descriptor; b: low word; hi: the descriptors' high word.
// KD 2: two blocks, the second one's M operand 1024 units further and its tokens at b2.
template <int CG, int H, bool TMEM_A, int KD>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t step, uint32_t a, uint32_t b, uint32_t b2, uint32_t hi,
                                          uint32_t idesc, uint32_t acc, uint32_t bar) {
    static_assert(KD == 1 || (H == 1 && !TMEM_A), "two blocks of one int8 tile");
    if constexpr (CG == 1 && KD == 2) PTQ8_BLOCK(PTQ8_D8("1") PTQ8_COMMIT1);
    if constexpr (CG == 2 && KD == 2) PTQ8_BLOCK(PTQ8_D8("2") PTQ8_COMMIT2);
    if constexpr (KD == 2) return;
    if constexpr (CG == 1 && H == 1 && !TMEM_A) PTQ8_BLOCK(PTQ8_S4("1") PTQ8_COMMIT1);
    if constexpr (CG == 1 && H == 2 && !TMEM_A) PTQ8_BLOCK(PTQ8_S8("1") PTQ8_COMMIT1);
    if constexpr (CG == 2 && H == 1 && !TMEM_A) PTQ8_BLOCK(PTQ8_S4("2") PTQ8_COMMIT2);
    if constexpr (CG == 2 && H == 2 && !TMEM_A) PTQ8_BLOCK(PTQ8_S8("2") PTQ8_COMMIT2);
    if constexpr (CG == 1 && H == 1 && TMEM_A) PTQ8_BLOCK(PTQ8_T4("1") PTQ8_COMMIT1);
    if constexpr (CG == 1 && H == 2 && TMEM_A) PTQ8_BLOCK(PTQ8_T8("1") PTQ8_COMMIT1);
    if constexpr (CG == 2 && H == 1 && TMEM_A) PTQ8_BLOCK(PTQ8_T4("2") PTQ8_COMMIT2);
    if constexpr (CG == 2 && H == 2 && TMEM_A) PTQ8_BLOCK(PTQ8_T8("2") PTQ8_COMMIT2);
}
#undef PTQ8_MMA
#undef PTQ8_S
#undef PTQ8_T
#undef PTQ8_S4
#undef PTQ8_S8
#undef PTQ8_D
#undef PTQ8_D8
#undef PTQ8_T4
#undef PTQ8_T8
#undef PTQ8_COMMIT1
#undef PTQ8_COMMIT2
#undef PTQ8_BLOCK

// Arrive on `bar` (the pair's: in both CTAs) when the MMAs issued so far have completed.
template <int CG>
__device__ __forceinline__ void commit_elect(uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred e;\n\t.reg .b16 m;\n\tmov.u16 m, 3;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}\n" ::"r"(bar)
            : "memory");
    else
        mma_commit_elect(bar);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16,"
        " %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[16]) { tmem_ld16(taddr, v); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void pin(uint32_t (&v)[16]) { pin_after(v); }
__device__ __forceinline__ void pin(uint32_t (&v)[8]) {
    asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]));
}
// One column; read through pinned() once it has been waited for.
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
    return v;
}
__device__ __forceinline__ int pinned(uint32_t v) {
    asm volatile("" : "+r"(v));
    return static_cast<int>(v);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- tiles

// Tile t of the launch: its group, first row, valid rows (0: none left) and channel tile.
// Order inside a group: bands of kBand token tiles; a band goes through the channel tiles with its
// token tiles innermost, so that CTAs running at the same time share both operands in L2.
struct Tile {
    int group, row0, valid, ct;
};
// Accumulator columns in use: as many as the tile has tokens, a multiple of 16 (of 32 for a pair).
template <int CG, int TN>
__device__ __forceinline__ int columns_of(const Tile& t) {
    return min(TN, (t.valid + 16 * CG - 1) / (16 * CG) * (16 * CG));
}

template <int TN>
struct Tiles {
    const LinearParams& l;
    const int* start;   // shared memory: first tile of each group, and the end; null: one group of all rows
    const int* row;     // and first row
    int ctiles;
    int g = 0;          // cursor: tiles are asked for in increasing order
    __device__ Tiles(const LinearParams& lp, const int* s, const int* r, int c) : l(lp), start(s), row(r), ctiles(c) {}
    __device__ bool get(int t, Tile& o) {
        int beg = 0, end = static_cast<int>(l.rows), i = t;
        if (start) {
            while (g < l.groups && t >= start[g + 1]) ++g;
            if (g >= l.groups) return false;
            beg = row[g];
            end = row[g + 1];
            i = t - start[g];
        }
        const int tt = (end - beg + TN - 1) / TN;   // rows + TN fits: the host limits rows
        if (!start && i >= tt * ctiles) return false;
        const int full = kBand * ctiles, band = i / full, rest = i - band * full;
        const int wide = min(kBand, tt - band * kBand);
        o.ct = rest / wide;
        const int k = band * kBand + (rest - o.ct * wide);
        o.group = g;
        o.row0 = beg + k * TN;
        o.valid = min(TN, end - o.row0);
        return true;
    }
};

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A lane's channel: scales and bias of the tile (two of each when gated).
template <int H>
struct Channel {
    float ws[H], b[H];
    bool ok;
};

template <int H>
__device__ __forceinline__ Channel<H> channel_of(const LinearParams& l, int group, int c) {
    Channel<H> ch;
    ch.ok = c < l.n;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const size_t at = static_cast<size_t>(group) * (l.n * H) + h * l.n + c;
        ch.ws[h] = ch.ok ? l.ws[at] : 0.0f;
        ch.b[h] = ch.ok && l.bias ? l.bias[at] : 0.0f;
    }
    return ch;
}

// A lane's outputs for two tokens, each step on both at once.  With SwiGLU: right where `most` stays below kSwigluMost.
template <int H, bool W4>
__device__ __forceinline__ float2 finish2(const Channel<H>& ch, float2 xs, const int2 (&a)[H], float2& most) {
    float2 v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        float2 acc = make_float2(__int2float_rn(a[h].x), __int2float_rn(a[h].y));
        if (W4) acc = __fmul2_rn(acc, both(0.0625f));   // the codes were multiplied as 16 times their value
        // dequant(); the last sum one by one, since the compiler fuses a packed product and sum
        acc = __fmul2_rn(acc, __fmul2_rn(xs, both(ch.ws[h])));
        v[h] = make_float2(__fadd_rn(acc.x, ch.b[h]), __fadd_rn(acc.y, ch.b[h]));
    }
    return H == 2 ? swiglu2(v[0], v[H - 1], most) : v[0];
}
// One output, whatever its gate.
template <bool W4>
__device__ __forceinline__ float finish_far(const Channel<2>& ch, float xs, int a0, int a1) {
    constexpr int shift = W4 ? 4 : 0;
    return swiglu(dequant(a0 >> shift, xs, ch.ws[0], ch.b[0]), dequant(a1 >> shift, xs, ch.ws[1], ch.b[1]));
}

// Columns [c0, c1) of a warp's 32 accumulator lanes -> y.  xs: shared address of their token scales, from column c0 on
// (zero past the end).
template <typename T, int H, bool W4, int TN>
__device__ __forceinline__ void store_columns(T* y, size_t ldy, uint32_t acc, uint32_t xs, const Channel<H>& ch, int c0, int c1) {
    // Columns at a time: eight where the unpackers leave few registers (4096 x 4096 -> 2 x 8192: 204 us, with sixteen 209).
    constexpr int N = W4 && H == 2 ? 8 : 16;
    for (int c = c0; c < c1; c += N, xs += 4 * N) {
        uint32_t v[N], u[N];
        tmem_ld(acc + c, v);
        if (H == 2) tmem_ld(acc + TN + c, u);
        tmem_wait_ld();
        pin(v);
        if (H == 2) pin(u);
        T* const out = y + static_cast<size_t>(c) * ldy;
        const int left = c1 - c;
        float2 most = both(0.0f);
        T* o = out;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 x4 = lds128f(xs + 4 * j);
#pragma unroll
            for (int i = j; i < j + 4; i += 2) {
                int2 a[H];
                a[0] = make_int2(v[i], v[i + 1]);
                if (H == 2) a[H - 1] = make_int2(u[i], u[i + 1]);
                const float2 r = finish2<H, W4>(ch, i & 2 ? make_float2(x4.z, x4.w) : make_float2(x4.x, x4.y), a, most);
                if (ch.ok && i < left) *o = from_f32<T>(r.x);
                o += ldy;
                if (ch.ok && i + 1 < left) *o = from_f32<T>(r.y);
                o += ldy;
            }
        }
        if constexpr (H == 2) {
            if (__any_sync(0xffffffffu, !(most.x + most.y < kSwigluMost))) {   // rare: once more, one by one
                o = out;
#pragma unroll 1
                for (int j = 0; j < min(left, N); ++j, o += ldy) {
                    const uint32_t g1 = tmem_ld1(acc + c + j), u1 = tmem_ld1(acc + TN + c + j);
                    tmem_wait_ld();
                    const float r = finish_far<W4>(ch, __int_as_float(lds32(xs + 4 * j)), pinned(g1), pinned(u1));
                    if (ch.ok) *o = from_f32<T>(r);
                }
            }
        }
    }
}

// The finishing half of a split tile: the S partial sums of this CTA's tokens, every step-th of them from `part`
// on, four at a time.  got: shared address of this lane's channel of the first token of the first CTA; a token is
// H * 128 bytes further, a CTA `cta` bytes.  xs: shared address of the scales of the tokens that this warp finishes.
template <typename T, int H, bool W4>
__device__ __forceinline__ void store_partials(T* y, size_t ldy, uint32_t got, int S, int cta, uint32_t xs, const Channel<H>& ch,
                                               int mine, int part, int step) {
    for (int t = part; t < mine; t += 4 * step, xs += 16) {
        int a[4][H] = {};
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)   // tokens past the end: what lies there is not used
#pragma unroll
                for (int h = 0; h < H; ++h) a[i][h] += lds32(got + s * cta + (min(t + i * step, mine - 1) * H + h) * 128);
        const float4 x4 = lds128f(xs);
        float2 most = both(0.0f);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            int2 b[H];
#pragma unroll
            for (int h = 0; h < H; ++h) b[h] = make_int2(a[i][h], a[i + 1][h]);
            const float2 r = finish2<H, W4>(ch, i ? make_float2(x4.z, x4.w) : make_float2(x4.x, x4.y), b, most);
            if (ch.ok && t + i * step < mine) y[static_cast<size_t>(t + i * step) * ldy] = from_f32<T>(r.x);
            if (ch.ok && t + (i + 1) * step < mine) y[static_cast<size_t>(t + (i + 1) * step) * ldy] = from_f32<T>(r.y);
        }
        if constexpr (H == 2) {
            if (!(most.x + most.y < kSwigluMost)) {   // rare: once more, one by one
#pragma unroll 1
                for (int i = t, k = 0; i < min(mine, t + 4 * step); i += step, ++k) {
                    int g1 = 0, u1 = 0;
                    for (int s = 0; s < S; ++s) {
                        g1 += lds32(got + s * cta + i * 256);
                        u1 += lds32(got + s * cta + i * 256 + 128);
                    }
                    const float r = finish_far<W4>(ch, __int_as_float(lds32(xs + 4 * k)), g1, u1);
                    if (ch.ok) y[static_cast<size_t>(i) * ldy] = from_f32<T>(r);
                }
            }
        }
    }
}

// 16 packed bytes -> 8 words of 16 times the 32 codes, in order.
__device__ __forceinline__ void widen(const uint4& p, uint32_t* o) {
    const uint32_t m = 0xF0F0F0F0u;
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t even = (w[i] << 4) & m, odd = w[i] & m;
        o[2 * i] = __byte_perm(even, odd, 0x5140);
        o[2 * i + 1] = __byte_perm(even, odd, 0x7362);
    }
}

template <int CG, int TN, bool W4, bool GATED>
__global__ void __launch_bounds__(TcShape<CG, TN, W4, GATED>::kThreads, TcShape<CG, TN, W4, GATED>::kPerSm)
    linear_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ TcParams p) {
    using Sh = TcShape<CG, TN, W4, GATED>;
    constexpr int H = Sh::H;
    extern __shared__ uint8_t dyn[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxLinStages + 14];
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float sxs_all[Sh::kEpi][Sh::kCW];   // token scales, each epilogue warp its own columns

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = CG == 1 ? p.split : 1;
    const bool clustered = CG == 2 || S > 1;
    const uint32_t rank = clustered ? cluster_rank() : 0;
    const bool leader = CG == 1 || rank == 0;

    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    uint8_t* const base_p = dyn + (base - smem_u32(dyn));
    const uint32_t after = base + p.stages * Sh::kStage;   // tile list, partial sums
    int* const list = reinterpret_cast<int*>(base_p + (after - base));   // first tile of each group, and the end
    int* const first_row = list + p.l.groups + 1;                        // and first row
    const uint32_t recv = after + p.list_bytes;
    const uint32_t b0 = smem_u32(bars);
    const uint32_t full = b0, empty = full + 8 * p.stages;
    const uint32_t afull = b0 + 8 * 2 * kMaxLinStages, accfull = afull + 64, accempty = accfull + 16,
                   partial = accempty + 16, drain = partial + 8;

    if (warp == 0 && elect_one()) {
        tma_prefetch(&map_x);
        tma_prefetch(&map_w);
    }
    if (warp == 1 && lane == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 8; ++a) mbar_init(afull + 8 * a, 4 * H * CG);
        for (int a = 0; a < 2; ++a) {
            mbar_init(accfull + 8 * a, 1);
            mbar_init(accempty + 8 * a, Sh::kEpi * CG);
        }
        mbar_init(partial, 1);
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 2) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                         "r"(p.tmem_cols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
            tmem_relinquish();
        }
    }
    const bool listed = p.l.offsets != nullptr;
    Tiles<TN> tiles(p.l, listed ? list : nullptr, first_row, p.ctiles);
    const int per = CG == 2 ? 2 : S;
    const int t0 = blockIdx.x / per, dt = gridDim.x / per;
    const int kb0 = static_cast<int>(static_cast<long long>(p.kblocks) * (S > 1 ? rank : 0) / S);
    const int kb1 = static_cast<int>(static_cast<long long>(p.kblocks) * (S > 1 ? rank + 1 : 1) / S);
    Tile tile;
    if (warp == 0 && !listed && tiles.get(t0, tile) && elect_one()) {
        // while the kernel before this one drains: the weights of the first stages
        const int c = (tile.ct * CG + static_cast<int>(CG == 2 ? rank : 0)) * 128;
        for (int kb = kb0 * Sh::KD; kb < min(kb1, kb0 + p.stages) * Sh::KD; ++kb)
            for (int h = 0; h < H; ++h) prefetch_3d(&map_w, kb * (W4 ? 64 : 128), h * p.l.n + c, 0);
    }
    __syncwarp();
    tc_fence_before();
    if (clustered) {   // the peers' barriers exist
        cluster_arrive_relaxed();
        cluster_wait();
    } else {
        __syncthreads();
    }
    // Only now, with this CTA's TMEM allocated, may the next kernel start: a CTA of it that took the columns first would wait
    // for this kernel, and this kernel's allocation, which has no limit, for that CTA.
    griddep_launch();
    griddep_wait();                  // nothing above reads or writes global memory (but for prefetches)
    if (listed && warp == 2) {
        // The groups' first rows, clamped into [0, rows] and never decreasing, then their first tiles: what the
        // offsets hold, the tiles are no more than the launch was made for.
        const int most = static_cast<int>(p.l.rows);
        int row = 0;
        for (int g0 = 0; g0 <= p.l.groups; g0 += 32) {
            int v = g0 + lane <= p.l.groups ? min(max(p.l.offsets[g0 + lane], 0), most) : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v = max(v, o);
            }
            v = max(v, row);
            if (g0 + lane <= p.l.groups) first_row[g0 + lane] = v;
            row = __shfl_sync(0xffffffffu, v, 31);
        }
        __syncwarp();
        int sum = 0;
        for (int g0 = 0; g0 < p.l.groups; g0 += 32) {
            int n = 0;
            if (g0 + lane < p.l.groups) n = (first_row[g0 + lane + 1] - first_row[g0 + lane] + TN - 1) / TN * p.ctiles;
            int incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            if (g0 + lane < p.l.groups) list[g0 + lane] = sum + incl - n;
            sum += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) list[p.l.groups] = sum;
    }
    __syncwarp();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, a_tiles = tmem + Sh::kACol0;

    const long long limit = p.wait_limit;
    bool arrived = false, failed = false;
    auto give_up = [&](int code) {
        failed = true;
        if (lane == 0) {
            *static_cast<volatile int*>(p.err) = code;
            __threadfence_system();
        }
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- producer
        // The pair's loads all count at the leader, which issues the MMAs; but packed weights at the own CTA, whose
        // unpackers read them.
        const uint32_t x_at = CG == 2 ? mapa(full, 0) : full, w_at = W4 ? full : x_at;
        int s = 0, issued = 0;
        uint32_t ph = 1;
        bool ok = true;
        for (int t = t0; ok && tiles.get(t, tile); t += dt) {
            const int c = (tile.ct * CG + static_cast<int>(CG == 2 ? rank : 0)) * 128;
            // the pair's MMA takes the first half of its columns from CTA 0, the other from CTA 1
            const int r = tile.row0 + (CG == 2 ? static_cast<int>(rank) * columns_of<CG, TN>(tile) / 2 : 0);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_warp(empty + 8 * s, ph, limit)) {
                    give_up(ERR_WAIT_EMPTY);
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    const uint32_t wdst = base + s * Sh::kStage, xdst = wdst + Sh::kW;
                    if (leader || W4) mbar_expect_tx(full + 8 * s, (W4 ? 1 : CG) * Sh::kW + (leader ? CG : 0) * Sh::kX);
                    if (!(p.stall && blockIdx.x == 0 && issued == 0)) {
#pragma unroll
                        for (int b = 0; b < Sh::KD; ++b) {
                            const int k = kb * Sh::KD + b;
#pragma unroll
                            for (int h = 0; h < H; ++h) {
                                if constexpr (W4)
                                    load_rows_3d<1>(wdst + h * 8192, &map_w, w_at + 8 * s, k * 64, h * p.l.n + c, tile.group);
                                else
                                    load_rows_3d<CG>(wdst + (b * H + h) * 16384, &map_w, w_at + 8 * s, k * 128, h * p.l.n + c,
                                                     tile.group);
                            }
                            load_rows_2d<CG>(xdst + b * Sh::kXBlock, &map_x, x_at + 8 * s, k * 128, r);
                        }
                    }
                }
                __syncwarp();
                ++issued;
                if (++s == p.stages) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (S > 1) break;
        }
        if (ok) {
            // every stage consumed: no commit is on its way to this CTA's barriers when it ends
            for (int i = 0; ok && i < p.stages; ++i) {
                ok = mbar_wait_warp(empty + 8 * s, ph, limit);
                if (++s == p.stages) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok) give_up(ERR_WAIT_EMPTY);
        }
        if (!ok) {
            // own copies in flight must land before the CTA ends (what a pair's second CTA loads counts at the leader, which
            // waits for it: no CTA ends before both have given up)
            const int n = min(issued, p.stages);
            for (int i = 1; i <= n; ++i) {
                const int back = issued - i;
                if (leader || W4) mbar_wait_warp(full + 8 * (back % p.stages), (back / p.stages) & 1, limit);
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer (the pair's leader)
        int s = 0, ab = 0, buf = 0;
        uint32_t ph = 0, aph = 0, accph = 1;
        const uint64_t desc = make_sdesc(base, 128);
        const uint32_t desc0 = static_cast<uint32_t>(desc), desc_hi = static_cast<uint32_t>(desc >> 32);
        bool ok = leader;
        for (int t = t0; ok && tiles.get(t, tile); t += dt) {
            const int nn = columns_of<CG, TN>(tile);
            const uint32_t idesc = (make_idesc_i8(nn) & ~(0x1Fu << 24)) | (static_cast<uint32_t>(128 * CG >> 4) << 24);
            const uint32_t d = tmem + buf * Sh::kCols;
            if (!mbar_wait_warp(accempty + 8 * buf, accph, limit)) {
                give_up(ERR_WAIT_ACC);
                ok = false;
                break;
            }
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb) {
                // W4: this CTA's unpackers saw the stage's loads arrive, the tokens' rows of both CTAs among them
                if (!mbar_wait_warp(W4 ? afull + 8 * ab : full + 8 * s, W4 ? aph : ph, limit)) {
                    give_up(ERR_WAIT_FULL);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t st = desc0 + s * (Sh::kStage >> 4);
                mma_block<CG, H, W4, Sh::KD>(d, TN, W4 ? a_tiles + ab * Sh::kACols : st, st + (Sh::kW >> 4),
                                             st + ((Sh::kW + Sh::kXBlock) >> 4), desc_hi, idesc, kb > kb0, empty + 8 * s);
                if (W4 && ++ab == Sh::kABufs) {
                    ab = 0;
                    aph ^= 1;
                }
                if (++s == p.stages) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok) break;
            commit_elect<CG>(accfull + 8 * buf);
            if (++buf == p.acc_bufs) {
                buf = 0;
                accph ^= 1;
            }
            if (S > 1) break;
        }
        if (leader && !ok) {   // MMAs in flight end before TMEM is freed
            if constexpr (CG == 1) {
                mma_commit_elect(drain);
                mbar_wait_warp(drain, 0, limit);
            } else {
                commit_elect<2>(drain);
                mbar_wait_warp(drain, 0, limit);
            }
        }
    } else if (warp >= 4 && warp < 4 + Sh::kEpi) {
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3, part = (warp - 4) >> 2;
        float* const sxs = sxs_all[warp - 4];
        const uint32_t xs_at = smem_u32(sxs);
        const int lane_c = quad * 32 + lane;
        const uint32_t accempty_at = CG == 2 ? mapa(accempty, 0) : accempty;
        int buf = 0;
        uint32_t accph = 0;
        for (int t = t0; tiles.get(t, tile); t += dt) {
            const int c = (tile.ct * CG + static_cast<int>(CG == 2 ? rank : 0)) * 128 + lane_c;
            const Channel<H> ch = channel_of<H>(p.l, tile.group, c);
            const int c0 = part * Sh::kCW, c1 = min(c0 + Sh::kCW, tile.valid);
            // split: this CTA's tokens of the tile
            const int tokens = TN / S, first = S > 1 ? static_cast<int>(rank) * tokens : 0, mine = min(max(tile.valid - first, 0), tokens);
            __syncwarp();
            if (S == 1) {
                for (int i = lane; i < (max(c1 - c0, 0) + 15) / 16 * 16; i += 32) sxs[i] = c0 + i < c1 ? p.l.xs[tile.row0 + c0 + i] : 0.0f;
            } else {   // of the tokens that this warp finishes
                constexpr int step = Sh::kEpi / 4;
                for (int t = part + lane * step; t < (mine + 4 * step - 1) / (4 * step) * 4 * step; t += 32 * step)
                    sxs[t / step] = t < mine ? p.l.xs[tile.row0 + first + t] : 0.0f;
            }
            __syncwarp();
            if (!mbar_wait_warp(accfull + 8 * buf, accph, limit)) {
                give_up(ERR_WAIT_ACC);
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * Sh::kCols + (static_cast<uint32_t>(quad * 32) << 16);
            const size_t at = static_cast<size_t>(tile.row0) * p.l.ldy + c;
            if (CG == 2 || S == 1) {
                if (p.l.y_type == Y_F32)
                    store_columns<float, H, W4, TN>(static_cast<float*>(p.l.y) + at, p.l.ldy, acc, xs_at, ch, c0, c1);
                else if (p.l.y_type == Y_F16)
                    store_columns<__half, H, W4, TN>(static_cast<__half*>(p.l.y) + at, p.l.ldy, acc, xs_at, ch, c0, c1);
                else
                    store_columns<__nv_bfloat16, H, W4, TN>(static_cast<__nv_bfloat16*>(p.l.y) + at, p.l.ldy, acc, xs_at, ch, c0, c1);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(accempty_at + 8 * buf);
                if (++buf == p.acc_bufs) {
                    buf = 0;
                    accph ^= 1;
                }
            } else {
                // Partial sums by receiver, then quadrant, token, tile: what this warp sends to one of them is one copy
                // from the stages' memory (every load into it has been used).  Storing single words to the peers
                // took 60 cycles a column.
                const int shift = 31 - __clz(tokens);   // S is a power of two
                const int piece = tokens * H * 128, slot = 4 * piece;   // bytes of a quadrant's sums, and of all
                if (warp == 4 && lane == 0) mbar_expect_tx(partial, S * mine * H * 512);
                for (int cc = c0; cc < c1; cc += 16) {
                    uint32_t v[H][16];
#pragma unroll
                    for (int h = 0; h < H; ++h) tmem_ld16(acc + h * TN + cc, v[h]);
                    tmem_wait_ld();
#pragma unroll
                    for (int h = 0; h < H; ++h) pin_after(v[h]);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {   // two tokens at least go to the same CTA
                        const int to = (cc + j) >> shift, tk = (cc + j) & (tokens - 1);
                        const uint32_t at_j = base + to * slot + quad * piece + tk * (H * 128) + lane * 4;
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            sts32(at_j + h * 128, v[h][j]);
                            sts32(at_j + (H + h) * 128, v[h][j + 1]);
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                const int to = (c0 >> shift) + lane, there = min(max(tile.valid - to * tokens, 0), tokens);
                if (to << shift < c0 + Sh::kCW && there > 0)
                    copy_to_peer(mapa(recv + rank * slot + quad * piece, to), base + to * slot + quad * piece, there * H * 128, mapa(partial, to));
                __syncwarp();
                const bool joined = mbar_wait_warp(partial, 0, limit);
                cluster_arrive_relaxed();   // what the peers sent here has left their memory
                arrived = true;
                if (!joined) {
                    give_up(ERR_WAIT_PARTIAL);
                    break;
                }
                const uint32_t got = recv + quad * piece + lane * 4;
                const size_t own = at + static_cast<size_t>(first) * p.l.ldy;
                constexpr int step = Sh::kEpi / 4;
                if (p.l.y_type == Y_F32)
                    store_partials<float, H, W4>(static_cast<float*>(p.l.y) + own, p.l.ldy, got, S, slot, xs_at, ch, mine, part, step);
                else if (p.l.y_type == Y_F16)
                    store_partials<__half, H, W4>(static_cast<__half*>(p.l.y) + own, p.l.ldy, got, S, slot, xs_at, ch, mine, part, step);
                else
                    store_partials<__nv_bfloat16, H, W4>(static_cast<__nv_bfloat16*>(p.l.y) + own, p.l.ldy, got, S, slot, xs_at, ch, mine, part, step);
                break;
            }
        }
    } else if (W4 && warp >= 4 + Sh::kEpi) {
        // ---------------------------------------------------------------- unpackers
        // Sets of four warps: gated, every other one works on the up tile; sets with the same tile take turns
        // at the blocks.  A block takes a set over 700 cycles from end to end, the MMAs 250 to 600.
        const int quad = warp & 3, set = (warp - 4 - Sh::kEpi) >> 2, row = quad * 32 + lane;
        const int half = GATED ? set & 1 : 0, first = GATED ? set >> 1 : set;
        const uint32_t afull_at = CG == 2 ? mapa(afull, 0) : afull;
        const uint32_t lanes = a_tiles + half * 32 + (static_cast<uint32_t>(quad * 32) << 16);
        const uint8_t* src = base_p + half * 8192 + row * 64;
        const int turn = (row >> 1) & 3;   // the 64-byte TMA swizzle of this row
        // This CTA's blocks, tile after tile.  Stages and operand tiles are multiples of the turns, so that each has
        // one set, which sees every phase of its barriers in order.  The operand tile of block i is free when block i - a_bufs is
        // released: its stage's barrier (its next phase cannot end before block i itself is unpacked).
        const int total = listed ? list[p.l.groups] : static_cast<int>((p.l.rows + TN - 1) / TN) * p.ctiles;
        const int tiles_here = t0 >= total ? 0 : S > 1 ? 1 : (total - t0 + dt - 1) / dt;
        const long long blocks = static_cast<long long>(tiles_here) * (kb1 - kb0);
        constexpr int step = Sh::kTurns;
        int s = first, ab = first, old = first;
        uint32_t ph = 0, oldph = 0;
        for (long long i = first; i < blocks; i += step) {
            if (!mbar_wait_warp(full + 8 * s, ph, limit)) {
                give_up(ERR_WAIT_UNPACK);
                break;
            }
            // all of the block in registers before the operand tile is free: what follows the MMAs'
            // release of it is the store alone
            uint32_t o[32];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                widen(*reinterpret_cast<const uint4*>(src + s * Sh::kStage + ((q ^ turn) << 4)), o + 8 * q);
            if (i >= Sh::kABufs) {
                if (!mbar_wait_warp(empty + 8 * old, oldph, limit)) {
                    give_up(ERR_WAIT_UNPACK);
                    break;
                }
                old += step;
                if (old >= p.stages) {
                    old -= p.stages;
                    oldph ^= 1;
                }
            }
            tc_fence_after();
            tmem_st32(lanes + ab * Sh::kACols, o);
            tmem_wait_st();
            tc_fence_before();
            // In the leader the arrival also passes on what the wait above saw: the tokens' rows.  From the second CTA it
            // stands for the TMEM stores alone.
            if (lane == 0) {
                if (leader)
                    mbar_arrive(afull + 8 * ab);
                else
                    mbar_arrive_cluster_relaxed(afull_at + 8 * ab);
            }
            ab += step;
            if (ab >= Sh::kABufs) ab -= Sh::kABufs;
            s += step;
            if (s >= p.stages) {
                s -= p.stages;
                ph ^= 1;
            }
        }
    }

    // No CTA of a cluster ends, and no TMEM is freed, while a peer may still reach it.  Partial sums sent by this
    // CTA have arrived when its peers have; if a wait for them ran out, the pause lets the copies land.
    __syncwarp();
    if (clustered && !arrived) cluster_arrive();
    if (clustered) cluster_wait();
    if (S > 1 && failed) {
        const long long c0 = clock64();
        while (clock64() - c0 < kLandCycles) {
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        if constexpr (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
        else
            tmem_dealloc(tmem, p.tmem_cols);
    }
}

}  // namespace ptq8

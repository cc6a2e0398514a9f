// PTX building blocks shared by the engine's conv kernels and the token operators:
// mbarriers with bounded waits, TMA loads, programmatic launch, tcgen05 (TMEM, kind::i8
// MMAs, descriptors) and int4 unpacking.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ptq8 {

// Codes a bounded wait that ran out records in its engine's device error word
// (an int in engine-owned device memory, passed to every kernel that waits, so
// one engine's timeout never aborts another engine's kernels).
enum : int {
    ERR_NONE = 0,
    ERR_WAIT_EMPTY = 1,
    ERR_WAIT_FULL = 2,
    ERR_WAIT_ACC = 3,
    ERR_DRAIN = 4,
};

// Default wait limit: about 2 s at the B200 boost clock; no wait in these
// kernels is expected to take more than microseconds.
constexpr long long kWaitLimitCycles = 4000000000LL;

// ------------------------------------------------------------------ PTX helpers

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void fence_mbar_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Arrive without release semantics.  The epilogue frees a TMEM accumulator
// this way: the only accesses to order are its tcgen05.ld reads (completed by
// tcgen05.wait::ld and ordered by tcgen05.fence::before_thread_sync); a release
// arrive would also wait for the warp's outstanding global stores to reach the
// point of coherence and put that latency on the MMA's critical path.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// One try of a phase wait.  (A suspend-time hint here, and a nanosleep back-off in
// mbar_wait, were both measured: neither changed a conv's time.)
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Bounded wait for the phase with the given parity to complete: false after
// `limit` clock cycles without completion.  The clock is read once per 8 tries
// (a try per clock read made the polling warps issue several times more
// instructions than the tries themselves).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, long long limit) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (mbar_try(bar, parity)) return true;
        if (clock64() - t0 > limit) return false;
    }
}

// The same wait by every lane of a converged warp; the result is made warp-uniform.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, long long limit) {
    const bool ok = mbar_wait(bar, parity, limit);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void tma_prefetch(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1,
                                            int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// Programmatic dependent launch: the forward's kernels are launched so that the
// next one may start while this one drains.  launch_dependents lets it be
// scheduled; wait blocks until every earlier kernel of the stream has completed
// and its memory is visible -- executed before the first read of anything an
// earlier kernel wrote.  (Both are no-ops without the launch attribute.)
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// D[tmem] (+)= A[smem desc] * B[smem desc]^T, signed int8 -> int32.
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One lane of a converged warp (elect.sync) issues the MMA.  The issuing warp
// runs its control loop with all 32 lanes: descriptors and counters stay
// warp-uniform, and the issue keeps its pace while the epilogue warps that
// share its scheduler are busy (a lone issuing lane inside a divergent branch
// issued N=64 MMAs several times slower under that load).
__device__ __forceinline__ void mma_i8_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The KS = CB/32 MMAs of one K chunk (K offsets 0, 32, 64, 96 bytes: descriptor
// start +2 per 32 bytes) in one asm block: one election and one accumulate
// predicate per chunk, one 64-bit add per further MMA.
template <int KS>
__device__ __forceinline__ void mma_chunk_elect(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    static_assert(KS == 1 || KS == 2 || KS == 4, "K chunk of 32, 64 or 128 bytes");
    if constexpr (KS == 1) {
        asm volatile(
            "{\n\t.reg .pred e, p;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(acc)
            : "memory");
    } else if constexpr (KS == 2) {
        asm volatile(
            "{\n\t.reg .pred e, p;\n\t.reg .b64 a1, b1;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "add.s64 a1, %1, 2;\n\t"
            "add.s64 b1, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], a1, b1, %3, 1;\n\t}\n" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(acc)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred e, p;\n\t.reg .b64 a1, b1, a2, b2, a3, b3;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "add.s64 a1, %1, 2;\n\t"
            "add.s64 b1, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], a1, b1, %3, 1;\n\t"
            "add.s64 a2, %1, 4;\n\t"
            "add.s64 b2, %2, 4;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], a2, b2, %3, 1;\n\t"
            "add.s64 a3, %1, 6;\n\t"
            "add.s64 b3, %2, 6;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::i8 [%0], a3, b3, %3, 1;\n\t}\n" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(acc)
            : "memory");
    }
}

__device__ __forceinline__ void mma_commit_elect(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar)
        : "memory");
}

// True in exactly one lane of the converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, e;\n\t}\n"
        : "=r"(pred));
    return pred != 0;
}

// Arrive on an mbarrier once every previously issued tcgen05.mma of this thread completes.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
        " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
          "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
          "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
          "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The same wait, naming the 16 registers of an earlier tmem_ld16 as read and written, so
// that the compiler keeps every use of them after it (a load whose wait comes later than
// the next instructions, issued ahead of the computation on the previous load).
// Compiler-ordering pins for the software-pipelined TMEM loads (no instruction is
// emitted): pin_after makes the computation on v start after the preceding asm
// statements (the next half's load issue); pin_before makes the values w be computed
// before the following asm statements (the wait for that load).
__device__ __forceinline__ void pin_after(uint32_t (&v)[16]) {
    asm volatile(""
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15]));
}
__device__ __forceinline__ void pin_before(const uint32_t (&w)[4]) {
    asm volatile("" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]));
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15])
                 :
                 : "memory");
}

// Shared-memory matrix descriptor for a K-major operand tile whose rows are
// `cb` bytes long and stored with the matching TMA swizzle (cb = 32/64/128):
// 8-row core groups `8*cb` bytes apart (SBO), LBO unused for swizzled K-major.
__device__ __forceinline__ uint64_t make_sdesc(uint32_t saddr, int cb) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>((8u * cb) >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;  // descriptor version for sm_100
    const uint64_t layout = cb == 128 ? 2u : (cb == 64 ? 4u : 6u);
    d |= layout << 61;
    return d;
}

// Instruction descriptor: kind::i8, D = s32, A = B = s8, both K-major, M = 128.
__host__ __device__ constexpr uint32_t make_idesc_i8(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(128 >> 4) << 24);
}

// Sign-extended int8 codes of the 8 int4 codes in packed word x (low nibble first):
// lo/hi = codes 8i+0..3 / 8i+4..7 as bytes.
__device__ __forceinline__ void unpack_w4(uint32_t x, uint32_t& lo, uint32_t& hi) {
    uint32_t a = x & 0x0F0F0F0Fu;          // codes 0, 2, 4, 6 (nibbles)
    uint32_t b = (x >> 4) & 0x0F0F0F0Fu;   // codes 1, 3, 5, 7
    a |= (a & 0x08080808u) * 0x1Eu;        // nibble bit 3 set -> byte 0xF0 | nibble (no carry between bytes)
    b |= (b & 0x08080808u) * 0x1Eu;
    lo = __byte_perm(a, b, 0x5140);        // a.b0 b.b0 a.b1 b.b1
    hi = __byte_perm(a, b, 0x7362);        // a.b2 b.b2 a.b3 b.b3
}

// Make this thread's generic-proxy shared-memory writes visible to the tensor core
// (async proxy) once the consumer has synchronised with it.
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void named_bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

}  // namespace ptq8

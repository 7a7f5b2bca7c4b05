// mbarriers with bounded waits and the tcgen05 instructions that the tensor-core kernels share (sm_100a).
#pragma once

#include "common.cuh"

namespace qb {

constexpr unsigned kWaitLimit = 1u << 22;
constexpr unsigned kSuspendHintNs = 20000;  // a waiting thread sleeps (up to this long) instead of spinning

__device__ __forceinline__ unsigned smem_u32(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint64_t* b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity), "r"(kSuspendHintNs)
        : "memory");
    return ok != 0;
}
// Bounded wait: false when it gave up after `limit` tries or another role aborted (then the caller unwinds).
__device__ __forceinline__ bool mbar_wait(uint64_t* b, unsigned parity, volatile int* abort_flag, unsigned* status,
                                          unsigned limit = kWaitLimit) {
    for (unsigned i = 0; i < limit; ++i) {
        if (mbar_try(b, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    set_error(status, ERR_WAIT_TIMEOUT);
    return false;
}

// The same bounded wait run by a whole warp: every lane polls and a vote makes the outcome warp-uniform (a lane that
// saw the phase complete polls again until all have; a completed phase keeps reading as complete until the barrier
// moves on, which needs this warp's own arrival).
__device__ __forceinline__ bool warp_wait(uint64_t* b, unsigned parity, volatile int* abort_flag, unsigned* status) {
    for (unsigned i = 0; i < kWaitLimit; ++i) {
        if (__all_sync(0xffffffffu, mbar_try(b, parity))) return true;
        if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
    *abort_flag = 1;
    set_error(status, ERR_WAIT_TIMEOUT);
    return false;
}

__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1 : 0), "r"(0), "r"(0), "r"(0), "r"(0)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// K-major operands in shared memory with rows of 128 or 64 bytes, swizzled (unswizzled ones were read several times slower):
// 16-byte chunk c of row r lies at sw_offset<ROW>(r, c); atoms of 8 rows follow each other.  The descriptor of K offset
// `bytes` (a multiple of 32) into the rows at addr (1024-byte aligned) is {sw_lo(addr + bytes), sw_hi<ROW>}.
template <int ROW>
__device__ __forceinline__ uint32_t sw_offset(int r, int c) {
    static_assert(ROW == 128 || ROW == 64, "bytes of a row");
    return uint32_t(r) * ROW + uint32_t(ROW == 128 ? c ^ (r & 7) : c ^ (r >> 1 & 3)) * 16;
}
__device__ __forceinline__ uint32_t sw_lo(uint32_t addr) { return (addr >> 4) & 0x3FFF | 1u << 16; }
template <int ROW>
constexpr uint32_t sw_hi = uint32_t(8 * ROW >> 4) | 1u << 14 | (ROW == 128 ? 2u : 4u) << 29;

// The MMAs on such operands: descriptors as their low words, the high ones constant.  The whole (converged) warp makes the
// call and one elected lane issues: with operands that the compiler knows to be the same in all lanes (warp_same) they go
// straight to uniform registers.  Issued by a branch on the lane, an MMA cost about 100 cycles of moving its operands.
template <uint32_t AHI, uint32_t BHI, uint32_t IDESC>
__device__ __forceinline__ void mma_i8_sw(uint32_t tmem_d, uint32_t a, uint32_t b, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %3, 0;\n\tmov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t@e tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %6, p;\n\t}" ::"r"(tmem_d), "r"(a), "r"(b), "r"(accumulate ? 1 : 0), "n"(AHI),
        "n"(BHI), "r"(IDESC)
        : "memory");
}
template <uint32_t AHI, uint32_t BHI, uint32_t IDESC>
__device__ __forceinline__ void mma_f16_sw(uint32_t tmem_d, uint32_t a, uint32_t b, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %3, 0;\n\tmov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %6, p;\n\t}" ::"r"(tmem_d), "r"(a), "r"(b), "r"(accumulate ? 1 : 0), "n"(AHI),
        "n"(BHI), "r"(IDESC)
        : "memory");
}
// mma_commit by one elected lane of the warp: the lane that issued the MMAs (the election is the same each time).
__device__ __forceinline__ void mma_commit_elect(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
// A value that all lanes hold alike, told to the compiler.
__device__ __forceinline__ int warp_same(int x) { return __shfl_sync(0xffffffffu, x, 0); }
// A in TMEM: lane = row, a 32-bit column holds two consecutive elements of K.
template <uint32_t BHI, uint32_t IDESC>
__device__ __forceinline__ void mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %3, 0;\n\tmov.b64 db, {%2, %4};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %5, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(accumulate ? 1 : 0),
        "n"(BHI), "r"(IDESC)
        : "memory");
}

// This thread's writes to shared memory become visible to the tensor cores and bulk copies.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t* base, uint32_t cols) {  // a whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

// TMEM -> registers: this warp's 32 lanes, N consecutive 32-bit columns from taddr (tmem_ld_wait before use).
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, int (&v)[N]) {
    static_assert(N == 2 || N == 4 || N == 8 || N == 16 || N == 32, "columns of a load");
    if constexpr (N == 2) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(taddr));
    } else if constexpr (N == 4) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(taddr));
    } else if constexpr (N == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(taddr));
    } else if constexpr (N == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
              "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
            : "r"(taddr));
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
            "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
              "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
              "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
              "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(taddr));
    }
}
// Orders the uses of a load's registers after the tmem_ld_wait before this call.
template <int N>
__device__ __forceinline__ void tmem_ready(int (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
// registers -> TMEM: this warp's 32 lanes, N consecutive columns from taddr (tmem_st_wait before others read them).
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const unsigned (&v)[N]) {
    static_assert(N == 8 || N == 16, "columns of a store");
    if constexpr (N == 8) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                     "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    } else {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
            "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
            "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
            : "memory");
    }
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

}  // namespace qb

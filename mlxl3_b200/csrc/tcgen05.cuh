// Tensor memory, tcgen05 products and the waits around them, for kernels whose CTA is the only one of its kind on the SM.
#pragma once

#include "common.cuh"

namespace b200exl3 {

__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_byte_addr) {
    // K-major operand, 128-byte swizzle: 8-row groups 1024 bytes apart, descriptor version 1
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_byte_addr & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;                 // leading byte offset (unused for swizzled K-major)
    d |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride byte offset
    d |= static_cast<uint64_t>(1) << 46;                 // version
    d |= static_cast<uint64_t>(2) << 61;                 // SWIZZLE_128B
    return d;
}

__device__ __forceinline__ void tmem_alloc(uint32_t* smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// One lane of a converged warp.  Products issued under `if (elect_one())` take 30 cycles each, under `if (lane == 0)` 68
// (128 x 16..64 tile, back to back): the first branch is known to be uniform, as the descriptors' registers want it.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// The same by the lanes for which `arrive` holds, without a branch; bar is a shared-memory address.
__device__ __forceinline__ void mbar_arrive(bool arrive, uint32_t bar) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %1, 0;\n@p mbarrier.arrive.shared::cta.b64 _, [%0];\n}"
                 ::"r"(bar), "r"(static_cast<uint32_t>(arrive)) : "memory");
}

// Wait that gives up after about a quarter of a second, or at once when another role of the CTA has
// already given up, so that a lost copy or a miscounted barrier ends the kernel instead of hanging it.
static __device__ __noinline__ bool qmm_wait_slow(uint64_t* bar, uint32_t parity, volatile int* cta_failed) {
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    constexpr uint32_t kNap = 20000;                             // the hardware wakes the thread when the phase completes
    const unsigned long long t0 = global_ns();
    while (true) {
        if (mbar_try_wait_for(bar, parity, kNap)) return true;
        if (*cta_failed || global_ns() - t0 > 250000000ull) { *cta_failed = 1; return false; }
    }
}
__device__ __forceinline__ bool qmm_wait(uint64_t* bar, uint32_t parity, volatile int* cta_failed) {
    return mbar_try_wait(bar, parity) || qmm_wait_slow(bar, parity, cta_failed);
}
// Copies and products that were still in flight when a wait gave up have to land before the CTA gives its memory back (as at the end of
// qmm_kernel).  Lanes leave the loop one by one: a warp barrier belongs behind it.
__device__ __forceinline__ void settle_after_failure(bool failed) {
    if (!failed) return;
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
}
// Barrier of some warps.  Not the aligned form (`bar.sync`), which all lanes of a warp have to execute as one: lanes come here
// from branches of their own (lane 0 from an atomic or an arrival), where nothing but a warp barrier brings them together again.
// The same holds for the instructions marked .sync.aligned -- allocation and release of tensor memory, its loads and stores and
// the waits for them: each has a warp barrier before it with no branch on the lane, no elected lane and no polling loop in
// between, and the branches around it are on values that all lanes share (warp, item, token counts).
__device__ __forceinline__ void group_sync(int id, int threads) {
    __syncwarp();
    asm volatile("barrier.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
    __syncwarp();
}

}  // namespace b200exl3
